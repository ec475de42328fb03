"""The prefill step behind a sliding window with sinks, against float64."""
import math

import pytest
import torch

from oracle import pool8_oracle as orc


def _vec(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rows(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


class Step:
    """Sequences (q_len, q_first, k_len, k_first) packed with a gap of two rows in front of each."""

    def __init__(self, seqs, Hq, Hkv, D, dtype, peers=1, seed=0):
        self.seqs, self.peers, self.dtype, self.Hkv = seqs, peers, dtype, Hkv
        self.q_start, self.k_start = [], []
        nq = nk = 0
        for ql, _, kl, _ in seqs:
            self.q_start.append(nq + 2), self.k_start.append(nk + 2)
            nq, nk = nq + ql + 2, nk + max(kl, 0) + 2
        self.q = _rows((nq, Hq, D), seed + 1, dtype)
        self.kv = _rows((nk + 1, 2 * Hkv, D), seed + 2, dtype)
        gap = torch.ones(nk + 1, dtype=torch.bool)
        for s, (_, _, kl, _) in zip(self.k_start, seqs):
            gap[s:s + max(kl, 0)] = False
        self.kv[gap] = math.nan  # rows of no sequence

    def run(self, lsa, window, sinks, o_dtype=None, lse=True, kv=None, **kw):
        q = self.q.cuda()
        kv = self.kv.cuda() if kv is None else kv
        o = torch.full(q.shape, 7.0, dtype=o_dtype or self.dtype, device="cuda")
        l = torch.full(q.shape[:2], 7.0, device="cuda") if lse else None
        col = lambda i: _vec([s[i] for s in self.seqs])  # noqa: E731
        lsa.window_attention_fwd(q, kv[:, :self.Hkv], kv[:, self.Hkv:], o, _vec(self.q_start), col(0), col(1), _vec(self.k_start), col(2), col(3),
                                 self.peers, max(s[0] for s in self.seqs), window, sinks, lse=l, **kw)
        return o, l

    def check(self, got, window, sinks):
        o, l = got[0].cpu(), got[1].cpu().double() if got[1] is not None else None
        named = torch.zeros(o.shape[0], dtype=torch.bool)
        half = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}[o.dtype]
        for (ql, qf, kl, kf), qs, ks in zip(self.seqs, self.q_start, self.k_start):
            kl = max(kl, 0)
            named[qs:qs + ql] = True
            want, lse, tol_o, tol_l = orc.prefill(self.q[qs:qs + ql], self.kv[ks:ks + kl, :self.Hkv], self.kv[ks:ks + kl, self.Hkv:], ql, qf, kl, kf,
                                                  self.peers, window, sinks)
            x = o[qs:qs + ql].double()
            assert torch.isfinite(x).all()
            assert ((x - want).abs() <= tol_o + half * (want.abs() + tol_o) + 2.0 ** -24).all(), ((x - want).abs() - tol_o).max()
            if l is not None:
                fin = torch.isfinite(lse)
                y = l[qs:qs + ql]
                assert torch.equal(fin, torch.isfinite(y)) and (y[~fin] == -math.inf).all() and ((y - lse).abs() <= tol_l)[fin].all()
        assert (o[~named] == 7).all() and (l is None or (l[~named] == 7).all())


DT = {"f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ CPU
def test_oracle_of_the_step():
    """The restatement against a loop over queries and keys."""
    q, k, v = (torch.randn(n, h, 8, dtype=torch.float64) for n, h in ((5, 4), (9, 2), (9, 2)))
    for window, sinks, peers, qf, kf in ((3, 1, 1, 4, 0), (2, 0, 1, 0, 0), (5, 3, 2, 9, 1), (1, 0, 3, 2, 0)):
        o, lse, _, _ = orc.prefill(q, k, v, 5, qf, 9, kf, peers, window, sinks)
        for m in range(5):
            qp = qf + m * peers
            seen = [n for n in range(9) if kf + n * peers <= qp and (qp - (kf + n * peers) < window or kf + n * peers < sinks)]
            for h in range(4):
                s = torch.stack([q[m, h] @ k[n, h // 2] / math.sqrt(8) for n in seen]) if seen else torch.empty(0)
                if not seen:
                    assert lse[m, h] == -math.inf and not o[m, h].any()
                else:
                    assert torch.allclose(lse[m, h], torch.logsumexp(s, 0)) and torch.allclose(o[m, h], torch.softmax(s, 0) @ torch.stack([v[n, h // 2] for n in seen]))


def test_library_refuses_bad_steps():
    import ctypes as C
    from loongserve_amd import _lib
    lib = _lib.load()

    def step(window=4, sinks=0, **kw):
        a = _lib.PrefillArgs(q=4096, k=4096, v=4096, q_stride_t=256, q_stride_h=128, k_stride_t=256, k_stride_h=128, v_stride_t=256, v_stride_h=128,
                             q_b_start_loc=4096, q_b_seq_len=4096, q_first_token_global_idx=4096, kv_b_start_loc=4096, kv_b_seq_len=4096,
                             kv_first_token_global_idx=4096, batch=0, num_q_heads=2, num_kv_heads=2, head_dim=128, dtype=0, sp_peers=1, max_q_len=4,
                             sm_scale=0.1, o=4096, o_stride_t=256, o_stride_h=128, o_dtype=0)
        for k, x in kw.items():
            setattr(a, k, x)
        return lib.lsattn_prefill_window(C.byref(a), window, sinks, None)
    assert step() == step(o_dtype=2) == step(window=1 << 60, sinks=1 << 60) == 0
    assert step(window=0) == step(sinks=-1) == step(o_dtype=1) == step(q=None) == step(sp_peers=0) == step(k_stride_t=4) == -1
    assert step(kv_cuts=2, kv_cut_len=64, o_cut_rows=8) == -1 and step(head_dim=48) == -2 and lib.lsattn_prefill_window(None, 4, 0, None) == -1


def test_python_operator_refuses():
    import loongserve_amd as lsa
    q, i = torch.zeros(4, 2, 128, dtype=torch.float16), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        lsa.window_attention_fwd(q, q, q, q, i, i, i, i, i, i, 1, 4, 8)


# ------------------------------------------------------------------------------------------------ GPU
@pytest.fixture(params=[None, "256"])
def rows(request, tuning):
    """The library's own shape, and 128-wide heads forced into that of 256 rows, which it keeps for larger launches."""
    tuning(prefill_rows=request.param)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (3, 3, 128), (4, 1, 64), (2, 2, 32), (6, 3, 16), (7, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 4), (64, 0), (100, 70), (1 << 40, 3)])
def test_prompts(lsa, rows, dtype, Hq, Hkv, D, window, sinks):
    s = Step([(n, 0, n, 0) for n in (1, 130, 0, 64, 301)], Hq, Hkv, D, DT[dtype], seed=Hq)
    s.check(s.run(lsa, window, sinks), window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("window,sinks", [(40, 0), (200, 5), (300, 129)])
def test_chunks_behind_contexts_shorter_and_later_keys_and_no_keys(lsa, rows, dtype, D, window, sinks):
    """A chunk at the end of its keys, one whose keys end before its window, one whose keys start behind its first queries, and one without keys."""
    s = Step([(50, 500, 550, 0), (20, 900, 300, 0), (90, 0, 60, 40), (5, 9, 0, 0), (33, 1000, 500, 533), (3, 5, -4, 0)], 4, 2, D, DT[dtype], seed=4)
    s.check(s.run(lsa, window, sinks), window, sinks)
    s.check(s.run(lsa, window, sinks, o_dtype=torch.float32), window, sinks)
    s.check(s.run(lsa, window, sinks, lse=False), window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Hq,Hkv,D,lens", [(32, 8, 128, [700, 333, 900]), (32, 32, 128, [400, 400]), (32, 4, 64, [900, 1000])])
def test_launches_that_fill_the_chip(lsa, rows, dtype, Hq, Hkv, D, lens):
    """Many workgroups: 32 positions per wave."""
    s = Step([(n, 0, n, 0) for n in lens] * (8 if D == 128 else 5), Hq, Hkv, D, DT[dtype], seed=6)
    s.seqs, keep = s.seqs, s.seqs
    for window, sinks in ((128, 4), (250, 0)):
        got = s.run(lsa, window, sinks)
        s.seqs = keep[:3]  # (the first few against float64; every other repeats their lengths)
        o = got[0].cpu()
        for (ql, qf, kl, kf), qs, ks in zip(s.seqs, s.q_start, s.k_start):
            want, lse, tol_o, tol_l = orc.prefill(s.q[qs:qs + ql], s.kv[ks:ks + kl, :Hkv], s.kv[ks:ks + kl, Hkv:], ql, qf, kl, kf, 1, window, sinks)
            half = 2.0 ** -11 if s.dtype == torch.float16 else 2.0 ** -8
            assert ((o[qs:qs + ql].double() - want).abs() <= tol_o + half * (want.abs() + tol_o) + 2.0 ** -24).all()
            assert ((got[1][qs:qs + ql].cpu().double() - lse).abs() <= tol_l).all()
        s.seqs = keep
        assert torch.isfinite(o.float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_a_ring_of_striped_chunks_joins_to_the_whole(lsa, rows, dtype):
    """Three instances hold every third token; the partials of one instance's queries over the three chunks merge to the step over all keys."""
    n, P, W, S = 300, 3, 70, 8
    q, kv = _rows((n, 4, 128), 1, DT[dtype]), _rows((n, 4, 128), 2, DT[dtype])
    want, lse, tol_o, tol_l = orc.prefill(q[1::P], kv[:, :2], kv[:, 2:], len(q[1::P]), 1, n, 0, 1, W, S)
    # (positions: query m of the instance is token 1 + 3 m)
    qp = 1 + 3 * torch.arange(len(q[1::P]))
    s = torch.einsum("mhd,nhd->mhn", q[1::P].double(), kv[:, :2].double().repeat_interleave(2, 1)) / math.sqrt(128)
    kp = torch.arange(n)
    seen = (kp[None] <= qp[:, None]) & ((kp[None] > qp[:, None] - W) | (kp[None] < S))
    s = s.masked_fill(~seen[:, None], -math.inf)
    want, lse = torch.einsum("mhn,nhd->mhd", torch.softmax(s, -1), kv[:, 2:].double().repeat_interleave(2, 1)), torch.logsumexp(s, -1)
    parts = []
    mine = q[1::P].contiguous().cuda()
    for r in range(P):
        rows = kv[r::P].contiguous().cuda()
        o, l = torch.empty(mine.shape, device="cuda"), torch.empty(mine.shape[:2], device="cuda")
        lsa.window_attention_fwd(mine, rows[:, :2], rows[:, 2:], o, _vec([0]), _vec([len(mine)]), _vec([1]), _vec([0]), _vec([len(rows)]), _vec([r]), P,
                                 len(mine), W, S, lse=l)
        parts.append((o, l))
    o, l = lsa.lse_merge(parts)
    assert ((o.cpu().double() - want).abs() <= tol_o.max() + 2.0 ** -20).all() and ((l.cpu().double() - lse).abs() <= tol_l.max() + 2.0 ** -20).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Hq,Hkv,window,sinks,seqs", [(4, 1, 900, 70, [(1200, 0, 1200, 0), (300, 2000, 2300, 0)]), (2, 2, 1500, 3, [(2100, 0, 2100, 0)]),
                                                      (1, 1, 640, 0, [(500, 1000, 1500, 0), (260, 700, 600, 100)]), (8, 1, 1100, 200, [(70, 3000, 3070, 0)])])
def test_windows_of_many_tiles(lsa, rows, dtype, Hq, Hkv, window, sinks, seqs):
    """Windows long enough for iterations without masks between those of the sinks, of the windows' starts and of the diagonal."""
    s = Step(seqs, Hq, Hkv, 128, DT[dtype], seed=10)
    # (scores that grow along the keys: the maximum is raised in every part of the walk)
    s.kv[:, :Hkv] *= torch.linspace(0.2, 3.0, s.kv.shape[0])[:, None, None].to(DT[dtype])
    s.check(s.run(lsa, window, sinks), window, sinks)
    s.check(s.run(lsa, window, sinks, o_dtype=torch.float32), window, sinks)


@pytest.mark.gpu
def test_far_positions(lsa, rows):
    """Positions close to 2^31, and a window wider than they are."""
    top = 2 ** 31 - 700
    s = Step([(40, top + 300, 340, top)], 4, 2, 128, torch.float16, seed=7)
    for window, sinks in ((50, 0), (50, 2 ** 31 - 600), (2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1)):
        s.check(s.run(lsa, window, sinks), window, sinks)


@pytest.mark.gpu
def test_strided_rows_a_stream_of_its_own_and_a_graph(lsa):
    s = Step([(200, 0, 200, 0), (61, 300, 361, 0)], 8, 2, 128, torch.float16, seed=8)
    wide = torch.full((s.kv.shape[0], 6, 160), 3.0, dtype=torch.float16, device="cuda")
    wide[:, 1:5, 16:144] = s.kv.cuda()
    s.check(s.run(lsa, 90, 3, kv=wide[:, 1:5, 16:144]), 90, 3)
    base = [t.clone() for t in s.run(lsa, 90, 3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = s.run(lsa, 90, 3)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, base))
    q, kv, o, l = s.q.cuda(), s.kv.cuda(), torch.empty_like(s.q, device="cuda"), torch.empty(s.q.shape[:2], device="cuda")
    vec = [_vec(s.q_start), _vec([200, 61]), _vec([0, 300]), _vec(s.k_start), _vec([200, 361]), _vec([0, 0])]
    call = lambda: lsa.window_attention_fwd(q, kv[:, :2], kv[:, 2:], o, *vec, 1, 200, 90, 3, lse=l)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in range(4):
        q.copy_(_rows(q.shape, seed, torch.float16))
        call()
        want = o.clone(), l.clone()
        o.zero_(), l.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o[2:202], want[0][2:202]) and torch.equal(l[2:202], want[1][2:202]) and torch.equal(o[204:], want[0][204:])


@pytest.mark.gpu
def test_refusals_on_the_gpu(lsa):
    q, i = torch.zeros(4, 2, 128, dtype=torch.float16, device="cuda"), _vec([0])
    call = lambda w=4, s=0, o=None, **kw: lsa.window_attention_fwd(q, q, q, torch.empty_like(q) if o is None else o, i, i, i, i, i, i, 1, 4, w, s, **kw)  # noqa: E731
    for bad in ((0, 0), (-1, 0), (4, -1), (None, 0)):
        with pytest.raises(ValueError, match="window"):
            call(*bad)
    with pytest.raises(ValueError, match="dtype of q"):
        call(o=torch.empty_like(q, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="lse"):
        call(lse=torch.empty(4, 3, device="cuda"))
    with pytest.raises(ValueError, match="shape of q"):
        call(o=torch.empty(4, 1, 128, dtype=torch.float16, device="cuda"))


@pytest.mark.gpu
def test_scores_of_keys_that_are_not_seen_do_not_matter(lsa, rows):
    """Infinities and NaN in K rows that no query sees, inside tiles that are walked."""
    s = Step([(300, 0, 300, 0)], 4, 2, 128, torch.float16, seed=9)
    ks = s.k_start[0]
    # (queries 200 .. 299 see keys 0, 1 and 151 .. 299)
    late = Step([(100, 200, 300, 0)], 4, 2, 128, torch.float16, seed=9)
    late.kv, late.k_start = s.kv.clone(), [ks]
    want = late.run(lsa, 50, 2)
    late.check(want, 50, 2)
    late.kv[ks + 2:ks + 151, 0] = math.inf
    late.kv[ks + 2:ks + 151, 1] = math.nan
    got = late.run(lsa, 50, 2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(256, 0), (300, 70), (1 << 40, 0)])
def test_waves_that_share_positions(lsa, dtype, D, window, sinks):
    """Launches of a workgroup per CU and less, two waves to a wave's positions: rows whose keys all lie in one wave's part, rows of none, a window that
    starts inside a part, lengths of zero and one."""
    s = Step([(301, 0, 301, 0), (1, 0, 1, 0), (0, 0, 0, 0), (17, 0, 17, 0), (40, 610, 650, 0), (33, 5, 20, 20), (9, 900, 400, 0)], 6, 2, D, DT[dtype], seed=12)
    s.kv[:, :2] *= torch.linspace(0.2, 3.0, s.kv.shape[0])[:, None, None].to(DT[dtype])
    s.check(s.run(lsa, window, sinks), window, sinks)
    s.check(s.run(lsa, window, sinks, o_dtype=torch.float32), window, sinks)
    s.check(s.run(lsa, window, sinks, lse=False), window, sinks)
