"""Requests that share tokens, at the ends: workspaces sized once, calls that are refused under way, requests freed twice, tables with holes, far positions."""
import math
import random

import pytest
import torch

from oracle import sharing_oracle as orc
from tests.test_gpu_sharing import DEV, F8, PAD, _case, _check, _decode_check, _decode_on_gpu, _i32, _prompt_case, _prompt_on_gpu, _rows

HEADS = [(32, 8, 128), (32, 32, 128), (28, 4, 64), (8, 1, 128), (7, 1, 64), (128, 64, 128), (2048, 1024, 64)]


# ------------------------------------------------------------------------------------------------ CPU: workspaces
@pytest.mark.parametrize("heads", HEADS)
def test_a_decode_workspace_for_the_largest_sizes_does_for_all(heads):
    """More requests, groups, prefix or own tokens never need less room: a program sizes one workspace for its longest steps."""
    from loongserve_amd import shared_prefix_decode_workspace_bytes as need
    rng = random.Random(heads[0])
    steps = ([1, 2, 4, 5, 16, 17, 32, 33, 64, 160, 161, 1000, 4096], [0, 1, 2, 3, 4, 12, 65, 200], [0, 1, 64, 65, 128, 1000, 16384, 131072],
             [0, 1, 32, 33, 64, 100, 128, 200, 513, 4000, 131072])
    for _ in range(3000):
        at = [rng.randrange(len(s)) for s in steps]
        sizes = [s[i] for s, i in zip(steps, at)]
        least = need(sizes[0], sizes[1], *heads, *sizes[2:])
        for k, s in enumerate(steps):
            if at[k] + 1 < len(s):
                more = sizes[:k] + [s[at[k] + 1]] + sizes[k + 1:]
                assert need(more[0], more[1], *heads, *more[2:]) >= least > 0, (sizes, more)


@pytest.mark.parametrize("heads", HEADS)
def test_a_prompt_workspace_for_the_most_rows_does_for_fewer(heads):
    """More rows or longer prefixes never need less room, whichever way either is taken."""
    from loongserve_amd import shared_prefix_attention_workspace_bytes as need
    prefixes = [1, 64, 65, 100, 6001, 131072]
    edges = sorted({1, 2, 3, 5, 100, 293, 5000, 65536} | {max(1, 98304 // heads[0] + d) for d in (-1, 0, 1)} | {g * 512 * heads[1] // heads[0] + d for g in (2, 12, 64) for d in (0, 1)})
    for groups in (1, 2, 12, 64, 500):
        for p, longer in zip(prefixes, prefixes[1:] + [200000]):
            for n, more in zip(edges, edges[1:] + [70000]):
                assert 0 < need(n, groups, *heads, p) <= min(need(more, groups, *heads, p), need(n, groups, *heads, longer)), (groups, p, n)


@pytest.mark.gpu
@pytest.mark.parametrize("own", [1, 100, 200, 2000])
def test_decode_steps_in_one_workspace(lsa, own):
    """Close bounds of the own tokens, from the first step to the last, in the workspace of the longest."""
    ws = torch.empty(lsa.shared_prefix_decode_workspace_bytes(64, 1, 32, 8, 128, 4000, 3000), dtype=torch.uint8, device=DEV)
    c = _case(51, 32, 8, 128, torch.float16, [(4000, [own] * 40)], [])
    got, want = _decode_on_gpu(lsa, c, workspace=ws), _decode_on_gpu(lsa, c)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ the prompts' step
def _prompt_some_rows(lsa, c, rows, what, eps_p=2.0 ** -11, **kw):
    """The step from the empty state against float64 at some of its rows; the outputs."""
    T, Hq, D = c["q"].shape
    kv, (start, size, req, pre) = c["kv"], c["g"]
    of = [max(g for g in range(len(start)) if start[g] <= i) for i in rows]
    want = [orc.prompt(c["q"][i:i + 1], kv[:, :c["Hkv"]], kv[:, c["Hkv"]:], c["table"], [0], [1], [req[g]], [pre[g]], c["most"], eps_p) for i, g in zip(rows, of)]
    o_ref, l_ref, tol_o, tol_l = (torch.cat(x) for x in zip(*want))
    o, m, l = torch.zeros(T, Hq, D, dtype=c["q"].dtype, device=DEV), torch.full((T, Hq), -math.inf, device=DEV), torch.zeros(T, Hq, device=DEV)
    _prompt_on_gpu(lsa, c, o, m, l, **kw)
    _check((o[rows], ((torch.log2(l) + m) * math.log(2))[rows]), (o_ref, l_ref, tol_o + orc.EPS_OUT[o.dtype] * (o_ref.abs() + tol_o) + 2.0 ** -25, tol_l + 1e-6), what)
    return o, m, l


@pytest.mark.gpu
def test_prompt_steps_in_one_workspace(lsa):
    """The workspace of the longest chunk for shorter ones, on either side of the rows from which a prefix is laid out."""
    heads = (128, 64, 128)
    ws = torch.empty(lsa.shared_prefix_attention_workspace_bytes(1500, 1, *heads, 300), dtype=torch.uint8, device=DEV)
    for rows in (1500, 768, 767, 100, 1):
        c = _prompt_case(53, *heads, torch.float16, [(300, rows)], tail=0)
        _prompt_some_rows(lsa, c, sorted({0, rows // 2, rows - 1}), rows, workspace=ws)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_step_without_the_room_to_lay_out(lsa, dtype):
    """A workspace for four groups, which are taken where they lie, and a call with one, which would be laid out if there were room."""
    heads, prefix, rows = (128, 64, 128), 4000, 800
    need = lsa.shared_prefix_attention_workspace_bytes
    small = torch.empty(need(rows, 4, *heads, prefix), dtype=torch.uint8, device=DEV)
    assert small.numel() < prefix * heads[1] * heads[2] * 4 <= need(rows, 1, *heads, prefix)
    c = _prompt_case(57, *heads, dtype, [(prefix, rows)], tail=0)
    looked_at = list(range(0, rows, 97)) + [rows - 1]
    guard = torch.full((small.numel() + 64,), 77, dtype=torch.uint8, device=DEV)
    _prompt_some_rows(lsa, c, looked_at, "where they lie", eps_p=orc.EPS_P[dtype], workspace=guard[:small.numel()])
    assert bool((guard[small.numel():] == 77).all())
    _prompt_some_rows(lsa, c, looked_at, "laid out")


@pytest.mark.gpu
def test_prompt_step_behind_a_loose_bound(lsa):
    """A bound far past the table's width costs no memory."""
    c = _prompt_case(59, 32, 8, 128, torch.float16, [(300, 3100)], tail=0)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    c["most"] = 1 << 22
    _prompt_some_rows(lsa, c, [0, 1700, 3099], "loose")
    assert torch.cuda.max_memory_allocated() - before < 1 << 30


# ------------------------------------------------------------------------------------------------ the managers
def _managers(lsa, slots=100, rows=6, width=40, dtype=torch.float16):
    mem = lsa.LongServeMemoryManager(slots, dtype, 2, 64, 3)
    return mem, lsa.LongServeReqManager(rows, width, mem)


def _request(lsa, mem, reqs, tokens):
    row, slots = reqs.alloc(1), mem.alloc(tokens)
    lsa.init_req_to_token_indexes(reqs.req_to_token_indexs, row.int(), _i32([tokens]), slots)
    return row, slots


def _as_counted(mem, reqs):
    assert mem.can_use_mem_size == int((mem.mem_state == 0).sum()) and reqs.can_use_req_size == int((reqs.req_state == 0).sum())


def _everything(mem, reqs):
    return [t.clone() for t in (mem.mem_state, reqs.req_state, reqs.req_to_token_indexs)] + [mem.can_use_mem_size, reqs.can_use_req_size]


def _same(a, b):
    return all(torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y for x, y in zip(a, b))


@pytest.mark.gpu
def test_requests_freed_twice_change_nothing(lsa):
    """A row that is free still names its old slots, which a fork may hold: freeing it again is refused, so is a row twice in a call, a row never taken."""
    mem, reqs = _managers(lsa)
    parent, slots = _request(lsa, mem, reqs, 20)
    other, _ = _request(lsa, mem, reqs, 7)
    fork = reqs.fork(parent, _i32([20]), 20)
    reqs.free_reqs(parent, _i32([20]), 20)
    assert mem.mem_state[slots].unique().tolist() == [1]
    before = _everything(mem, reqs)
    unused = torch.tensor([4], device=DEV)
    for rows, lens in ((parent, [20]), (torch.cat([other, parent]), [7, 20]), (other.repeat(2), [7, 7]), (unused, [0]), (torch.cat([fork, other, fork]), [20, 7, 0])):
        with pytest.raises(IndexError, match="request"):
            reqs.free_reqs(rows, _i32(lens), 20)
        assert _same(before, _everything(mem, reqs))
    for rows, lens in ((fork, _i32([20, 1])), (fork, _i32([20]).float())):
        with pytest.raises(ValueError):
            reqs.free_reqs(rows, lens, 20)
        assert _same(before, _everything(mem, reqs))
    reqs.free_reqs(torch.cat([other, fork]).int(), _i32([7, 20]), 20)
    _as_counted(mem, reqs)
    assert mem.can_use_mem_size == 100 and reqs.can_use_req_size == 6
    reqs.free_reqs(fork[:0], _i32([]), 20)


@pytest.mark.gpu
def test_requests_outside_the_table_are_refused(lsa):
    mem, reqs = _managers(lsa)
    row, _ = _request(lsa, mem, reqs, 5)
    before = _everything(mem, reqs)
    for bad in (-1, 6, 1 << 20, 1 << 40):
        with pytest.raises(IndexError, match="request"):
            reqs.free_reqs(torch.cat([row, torch.tensor([bad], device=DEV)]), _i32([5, 0]), 20)
        assert _same(before, _everything(mem, reqs))


@pytest.mark.gpu
def test_tokens_that_were_gone_leave_the_counts_right(lsa):
    """A live request some of whose tokens were freed one by one: an IndexError, everything else is freed, the counts fit."""
    mem, reqs = _managers(lsa)
    row, slots = _request(lsa, mem, reqs, 20)
    mem.free(slots[15:])
    with pytest.raises(IndexError, match="5 tokens"):
        reqs.free_reqs(row, _i32([20]), 20)
    _as_counted(mem, reqs)
    assert mem.can_use_mem_size == 100 and reqs.can_use_req_size == 6


@pytest.mark.gpu
def test_forks_that_are_refused_take_nothing(lsa):
    mem, reqs = _managers(lsa)
    row, _ = _request(lsa, mem, reqs, 20)
    before = _everything(mem, reqs)
    two = row.repeat(2)
    for lens, most in ((_i32([20]), 20), (_i32([20, 20]).float(), 20), (_i32([20, 20]).cpu(), 20), (_i32([20, 20]), -1), (_i32([[20, 20]]), 20)):
        with pytest.raises(ValueError):
            reqs.fork(two, lens, most)
        assert _same(before, _everything(mem, reqs))
        with pytest.raises(ValueError):
            reqs.fork_copy(two, lens, most, 40)
        assert _same(before, _everything(mem, reqs))
    with pytest.raises(AssertionError):
        reqs.fork_copy(two, _i32([20, 20]), 20, 81)  # more than the pool has
    assert _same(before, _everything(mem, reqs))


@pytest.mark.gpu
def test_forks_do_not_take_up_slots_that_are_free(lsa):
    """Entries behind a request's tokens may name slots that are free: nobody holds them, and a fork does not either."""
    mem, reqs = _managers(lsa)
    row, slots = _request(lsa, mem, reqs, 20)
    mem.free(slots[12:18].contiguous())
    forks = reqs.fork(row.repeat(3), _i32([20, 14, 12]), 20)
    _as_counted(mem, reqs)
    table = reqs.req_to_token_indexs.cpu()
    held = slots.int().tolist()
    held[12:18] = [PAD] * 6
    for f, n in zip(forks.tolist(), (20, 14, 12)):
        assert table[f, :n].tolist() == held[:n]
    assert table[int(row), :20].tolist() == slots.tolist()  # the source's own entries stay
    assert mem.mem_state[slots].tolist() == [4] * 12 + [0] * 6 + [2] * 2


@pytest.mark.gpu
def test_forks_and_copies_of_no_request(lsa):
    """Positions that get no slot name none: a row's entries from before are other requests' by now."""
    for copies in (False, True):
        table = torch.arange(80, dtype=torch.int32, device=DEV).reshape(8, 10).contiguous()
        state = torch.ones(100, dtype=torch.int32, device=DEV)
        src, dst, lens = _i32([-1, 8, 1, 1, 1, 1, 1]), _i32([2, 3, 4, 5, 6, 7, 99]), _i32([4, 10, 3, 10, 0, 25, 5])
        want = table.cpu().clone()
        want[2, :4] = PAD
        want[3, :] = PAD
        if copies:
            pool = torch.arange(2 * 100 * 2 * 64, device=DEV).reshape(2, 100, 2, 64).half()
            rows = pool.cpu().clone()
            index = torch.arange(80, 100, device=DEV)
            start = [0, 4, 0, 3, 0, 13, 0]  # 20 slots: the last request of 10 has 7 of them
            index[5] = 100  # and one that does not exist, of the second one's
            lsa.copy_requests(table, src, dst, lens, _i32(start), 10, index, pool)
            for s, n, at in ((4, 3, 0), (5, 10, 3), (7, 10, 13)):
                for i in range(n):
                    new = int(index[at + i]) if at + i < 20 else 100
                    want[s, i] = new if new < 100 else PAD
                    if new < 100:
                        rows[:, new] = rows[:, 10 + i]
            assert torch.equal(pool.cpu(), rows)
        else:
            lsa.fork_requests(table, src, dst, lens, 10, state)
            want[4, :3], want[5], want[7] = want[1, :3].clone(), want[1].clone(), want[1].clone()
            held = torch.ones(100, dtype=torch.int32)
            held[10:20] += 2
            held[10:13] += 1
            assert torch.equal(state.cpu(), held)
        assert torch.equal(table.cpu(), want), copies


@pytest.mark.gpu
def test_copies_are_whole_or_refused(lsa):
    """fork_copy refuses a source with positions that have no slot, and a total that is less than the tokens: nothing is taken."""
    mem, reqs = _managers(lsa)
    row, slots = _request(lsa, mem, reqs, 20)
    before = _everything(mem, reqs)
    for total in (0, 39):
        with pytest.raises(ValueError, match="total_len"):
            reqs.fork_copy(row.repeat(2), _i32([20, 20]), 20, total)
        assert _same(before, _everything(mem, reqs))
    for lens in ([21], [400]):
        with pytest.raises(ValueError, match="no slot"):
            reqs.fork_copy(row, _i32(lens), 400, 41)
        assert _same(before, _everything(mem, reqs))
    with pytest.raises(ValueError, match="no slot"):
        reqs.fork_copy(torch.tensor([6], device=DEV), _i32([3]), 20, 3)
    assert _same(before, _everything(mem, reqs))
    mem.free(slots[7:8])
    before = _everything(mem, reqs)
    with pytest.raises(ValueError, match="1 positions"):
        reqs.fork_copy(row, _i32([20]), 20, 20)
    assert _same(before, _everything(mem, reqs))
    mem.add_refs(slots[7:8])
    new, own = reqs.fork_copy(row.repeat(3), _i32([20, -5, 400]), 20, 41)  # (cut at 20 positions; a slot to spare)
    assert len(own) == 41 and torch.equal(reqs.req_to_token_indexs[new[0], :20].long(), own[:20]) and torch.equal(reqs.req_to_token_indexs[new[2], :20].long(), own[20:40])
    assert torch.equal(mem.kv_buffer[:, own[20:40]].view(torch.int16), mem.kv_buffer[:, slots].view(torch.int16))
    _as_counted(mem, reqs)


# ------------------------------------------------------------------------------------------------ far positions
@pytest.mark.gpu
def test_positions_past_a_billion(lsa):
    """Byte offsets in a table's row that pass 32 bits: a prefix of 2^30 positions and more, of which a few exist, in both attention operators."""
    far, D = 1 << 30, 64
    P = far + 70
    g = torch.Generator().manual_seed(61)
    kv, q = _rows((60, 2, D), g, torch.float16), _rows((3, 8, D), g, torch.float16)
    table = torch.full((3, P + 5), -1, dtype=torch.int32, device=DEV)
    near = {7: 1, far // 2 + 3: 2}
    there = {**near, **{far + i: 3 + i for i in range(40)}, P - 1: 50}
    for pos, slot in there.items():
        table[1, pos] = slot
    table[0, P:P + 5], table[2, P:P + 2] = _i32([51, 52, 53, 54, 55]), _i32([56, 57])
    kv_gpu = kv.to(DEV)
    o, lse = lsa.longserve_shared_prefix_decode_attention(q[:2].to(DEV), table, _i32([0, 2]), _i32([P + 5, P + 2]), 5, kv_gpu[:, :1], kv_gpu[:, 1:], _i32([0]), _i32([2]), _i32([1]),
                                                          _i32([P]), P, max_own_len=5)
    small = torch.full((3, len(there) + 5), PAD, dtype=torch.int32)
    n = len(there)
    small[1, :n] = torch.tensor(list(there.values()))
    small[0, n:n + 5], small[2, n:n + 2] = torch.arange(51, 56), torch.arange(56, 58)
    _check((o, lse), orc.decode(q[:2], kv[:, :1], kv[:, 1:], small, torch.tensor([0, 2]), torch.tensor([n + 5, n + 2]), [0], [2], [1], [n], n, torch.float16), "decode")
    o, m, l = torch.zeros(3, 8, D, dtype=torch.float16, device=DEV), torch.full((3, 8), -math.inf, device=DEV), torch.zeros(3, 8, device=DEV)
    lsa.shared_prefix_attention_fwd(q.to(DEV), kv_gpu[:, :1], kv_gpu[:, 1:], o, _i32([0]), _i32([3]), table, _i32([1]), _i32([P]), 3, P, m, l)
    o_ref, l_ref, tol_o, tol_l = orc.prompt(q, kv[:, :1], kv[:, 1:], small, [0], [3], [1], [n], n, 2.0 ** -11)
    _check((o, (torch.log2(l) + m) * math.log(2)), (o_ref, l_ref, tol_o + 2.0 ** -11 * (o_ref.abs() + tol_o) + 2.0 ** -25, tol_l + 1e-6), "prompt")


# ------------------------------------------------------------------------------------------------ the weights' bits
BITS = {"one": ([(200, [1, 33, 64, 7])], []), "long": ([(1000, [100] * 5), (513, [0] * 3)], []), "rows-past-a-tile": ([(130, [2] * 37)], [9, 1]),
        "tile-ends": ([(63, [3]), (64, [0, 5]), (65, [32, 31, 1]), (128, [1])], [1, 40])}


def _even(c):
    """The same case with small scores and V of one size: what a sum of products may be off by grows with them, and would hide the weights' bits."""
    c["q"] = (c["q"].float() / 64).to(c["q"].dtype)
    c["kv"][:, c["Hkv"]:] = c["kv"][:, c["Hkv"]:].clamp(-1, 1)
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(8, 2, 128), (16, 1, 128), (20, 2, 64)])
@pytest.mark.parametrize("name", list(BITS))
def test_decode_weights_in_float32_outputs(lsa, name, heads, dtype):
    """What the weights over a prefix are off by, where the output's rounding does not hide it: 2^-11 (fp16), 2^-16 (two parts of bfloat16)."""
    groups, alone = BITS[name]
    c = _even(_case(71, *heads, dtype, groups, alone))
    _decode_check(lsa, c, (name, heads, dtype), out_dtype=torch.float32, out=torch.empty(c["q"].shape, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(8, 2, 128), (7, 1, 128), (4, 4, 64)])
@pytest.mark.parametrize("groups", [[(500, 40), (3, 90)], [(2000, 300)], [(90, 5)] * 3])
def test_prompt_weights_of_bfloat16_rows(lsa, heads, groups):
    """Rows that are taken where they lie: P in two parts.  (O is the mean of hundreds of values of either sign: where it is small, its rounding does not hide the weights'.)"""
    c = _even(_prompt_case(73, *heads, torch.bfloat16, groups, tail=0))
    rows = len(c["q"])
    assert rows * heads[0] < 98304
    _prompt_some_rows(lsa, c, sorted(set(range(0, rows, 7)) | {rows - 1}), (heads, groups), eps_p=orc.EPS_P[torch.bfloat16])


def test_the_weights_bits_would_be_missed():
    """The two tests above see a kernel that keeps one part of a bfloat16 weight: planted in the oracle's weights, it is past their tolerances."""
    one_part = lambda p: (p * 512).bfloat16().double() / 512  # noqa: E731  (the largest is 2^9 there)

    def off(q, k, v, out_dtype):
        o, lse, tol, _ = orc.attend(q, k, v, orc.EPS_P[torch.bfloat16])
        s = torch.einsum("mhd,nhd->mhn", q.double(), k.double().repeat_interleave(q.shape[1] // k.shape[1], 1)) / math.sqrt(q.shape[2])
        p = torch.exp(s - s.amax(-1, keepdim=True))
        planted = torch.einsum("mhn,nhd->mhd", one_part(p), v.double().repeat_interleave(q.shape[1] // v.shape[1], 1)) / p.sum(-1, keepdim=True)
        tol = tol + orc.EPS_OUT[out_dtype] * (o.abs() + tol) + 2.0 ** -25
        return float(((planted.to(out_dtype).double() - o).abs() / tol).max())
    c = _even(_case(71, 8, 2, 128, torch.bfloat16, *BITS["rows-past-a-tile"]))
    slots = c["table"][c["g"][2][0], :130].long()
    assert off(c["q"][:37], c["kv"][slots, :2], c["kv"][slots, 2:], torch.float32) > 2
    c = _even(_prompt_case(73, 8, 2, 128, torch.bfloat16, [(500, 40), (3, 90)], tail=0))
    slots = c["table"][c["g"][2][0], :500].long()
    assert off(c["q"][:40], c["kv"][slots, :2], c["kv"][slots, 2:], torch.bfloat16) > 2


# ------------------------------------------------------------------------------------------------ pools of other sizes and types, other streams
@pytest.mark.gpu
@pytest.mark.parametrize("rows, slots", [(40, 700_000), (800, 700_000), (800, 2_200_000)])
def test_prompts_of_slots_past_two_gigabytes(lsa, rows, slots):
    """Offsets of slots that pass 31 and 32 bits, prefixes where they lie and laid out."""
    Hq, Hkv, D = (128, 16, 128) if rows > 100 else (32, 16, 128)
    pool = torch.empty(slots, 2 * Hkv, D, dtype=torch.float16, device=DEV)
    assert pool.numel() * 2 > (1 << 32) and slots * 2 * Hkv * D * 2 > 2 ** 31
    c = _prompt_case(79, Hq, Hkv, D, torch.float16, [(300, rows)], tail=0)
    far = torch.randperm(slots, generator=c["gen"])[:len(c["kv"])].sort().values
    far[-5:] = torch.arange(slots - 5, slots)
    assert len(far.unique()) == len(far)
    pool[far.to(DEV)] = c["kv"].to(DEV)
    t = c["table"]
    table = torch.where((t >= 0) & (t < len(far)), far[t.clamp(0, len(far) - 1).long()].int(), t)
    o, m, l = torch.zeros(rows, Hq, D, dtype=torch.float16, device=DEV), torch.full((rows, Hq), -math.inf, device=DEV), torch.zeros(rows, Hq, device=DEV)
    s, n, r, p = (_i32(x) for x in c["g"])
    lsa.shared_prefix_attention_fwd(c["q"].to(DEV), pool[:, :Hkv], pool[:, Hkv:], o, s, n, table.to(DEV), r, p, rows, 300, m, l)
    i = sorted({0, rows // 3, rows - 1})
    o_ref, l_ref, tol_o, tol_l = orc.prompt(c["q"][i], c["kv"][:, :Hkv], c["kv"][:, Hkv:], t, [0], [len(i)], c["g"][2], c["g"][3], 300, 2.0 ** -11)
    _check((o[i], (torch.log2(l[i]) + m[i]) * math.log(2)), (o_ref, l_ref, tol_o + 2.0 ** -11 * (o_ref.abs() + tol_o) + 2.0 ** -25, tol_l + 1e-6), (rows, slots))


@pytest.mark.gpu
def test_all_of_it_on_another_stream(lsa):
    """Prompts both ways, forks, copies, releases and compaction behind work that is queued on their stream."""
    side = torch.cuda.Stream()
    for heads, rows in (((8, 2, 128), 30), ((128, 64, 128), 800)):
        c = _prompt_case(83, *heads, torch.float16, [(200, rows)], tail=0)
        T, Hq, D = c["q"].shape
        kv, q, s = c["kv"].to(DEV), c["q"].to(DEV), [_i32(x) for x in c["g"]]
        table, late = c["table"].to(DEV), torch.zeros_like(kv)
        out = []
        for stream, pool in ((torch.cuda.current_stream(), kv), (side, late)):
            o, m, l = torch.zeros_like(q), torch.full((T, Hq), -math.inf, device=DEV), torch.zeros(T, Hq, device=DEV)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                if pool is late:
                    torch.cuda._sleep(20_000_000)
                    late.copy_(kv)
                lsa.shared_prefix_attention_fwd(q, pool[:, :c["Hkv"]], pool[:, c["Hkv"]:], o, s[0], s[1], table, s[2], s[3], rows, 200, m, l)
            stream.synchronize()
            out.append((o, m, l))
        assert all(torch.equal(a, b) for a, b in zip(*out))
    table0 = torch.full((6, 30), PAD, dtype=torch.int32)
    table0[0] = torch.randperm(200, generator=torch.Generator().manual_seed(4))[:30].int() + 100
    rows0 = torch.randn(2, 300, 4, 64).half()
    state0 = torch.zeros(300, dtype=torch.int32)
    state0[table0[0].long()] = 1
    free = torch.arange(0, 30)
    out = []
    for stream in (torch.cuda.current_stream(), side):
        table, pool, state = torch.zeros(6, 30, dtype=torch.int32, device=DEV), torch.zeros(2, 300, 4, 64, dtype=torch.float16, device=DEV), torch.zeros(300, dtype=torch.int32, device=DEV)
        now = [x.to(DEV) for x in (table0, rows0, state0, free)]
        zero, one, two, n = _i32([0]), _i32([1]), _i32([2]), _i32([30])
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(20_000_000)
            for x, y in zip((table, pool, state), now):
                x.copy_(y)
            lsa.fork_requests(table, zero, one, n, 30, state)
            state[now[3]] += 1
            lsa.copy_requests(table, zero, two, n, zero, 30, now[3], pool)
            freed = lsa.release_requests(table, _i32([0, 1]), _i32([30, 12]), 30, state)
            remap = lsa.compact_pool(state, pool, table, _i32([1, 2]), _i32([30, 30]), 30)
        stream.synchronize()
        out.append((table, pool, state, remap, freed))
    assert out[0][4] == out[1][4] == 12 and all(torch.equal(a, b) for a, b in zip(out[0][:4], out[1][:4]))
    table, pool, state = out[1][0].cpu(), out[1][1].cpu(), out[1][2].cpu()
    held = table0[0].long()
    assert torch.equal(pool[:, table[2].long()], rows0[:, held]) and torch.equal(pool[:, table[1, 12:].long()], rows0[:, held[12:]])
    assert state[:48].tolist() == [1] * 48 and not bool(state[48:].any())


@pytest.mark.gpu
@pytest.mark.parametrize("size", [300, 70000])
def test_compaction_without_rows(lsa, size):
    """The entry point of the library with no rows to move: counts, table and remap alone."""
    import ctypes as C
    from loongserve_amd import _lib
    lib, g = _lib.load(), torch.Generator().manual_seed(size)
    state = (torch.rand(size, generator=g) < 0.4).int() * 3
    used = state.nonzero().squeeze(1)
    table = used[torch.randint(0, len(used), (3, 50), generator=g)].int()
    table[1, 3] = PAD
    want_s, want_t, want_r, _, _ = orc.compact(state, table, [2, 0], [50, 20], 50)
    st, t, remap = state.to(DEV), table.to(DEV), torch.empty(size, dtype=torch.int32, device=DEV)
    req, lens, ws = _i32([2, 0]), _i32([50, 20]), torch.empty(lib.lsattn_compact_workspace_bytes(size), dtype=torch.uint8, device=DEV)
    a = _lib.CompactArgs(mem_state=st.data_ptr(), pool_size=size, remap=remap.data_ptr(), req_to_tokens=t.data_ptr(), num_reqs=3, max_seq_len=50, b_req_idx=req.data_ptr(),
                         b_seq_len=lens.data_ptr(), n=2, max_len_in_batch=50, workspace=ws.data_ptr(), workspace_bytes=ws.numel())
    assert lib.lsattn_compact_pool(C.byref(a), C.byref(_lib.PoolRows()), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(st.cpu(), want_s) and torch.equal(t.cpu(), want_t) and torch.equal(remap.cpu(), want_r)


@pytest.mark.gpu
def test_managers_of_an_8_bit_pool(lsa):
    """Forks, copies and compaction of a pool in 8 bits: rows and exponents together, read back bit for bit; decode over the copies."""
    mem, reqs = _managers(lsa, slots=200, dtype=F8)
    g = torch.Generator().manual_seed(89)
    gap = mem.alloc(30)
    row, slots = _request(lsa, mem, reqs, 33)
    src = torch.randn(33, 4, 64, generator=g).half().to(DEV)
    for layer in range(3):
        lsa.kv_scatter_fp8(src * 2.0 ** layer, slots, mem.kv_buffer[layer], mem.kv_scales[layer])

    def read(r):
        out = torch.zeros(3, 33, 4, 64, dtype=torch.float16, device=DEV)
        for layer in range(3):
            lsa.kv_gather_fp8(mem.kv_buffer[layer], mem.kv_scales[layer], reqs.req_to_token_indexs, r.int(), _i32([33]), _i32([0]), 33, out[layer])
        return out
    want = read(row)
    assert float((want[2] - src * 4).abs().max()) <= 2.0 ** -4 * float((src * 4).abs().max())
    fork = reqs.fork(row, _i32([33]), 33)
    copy, own = reqs.fork_copy(fork, _i32([33]), 33, 33)
    mem.free(gap)
    reqs.free_reqs(row, _i32([33]), 33)
    remap = mem.compact(reqs.req_to_token_indexs, torch.cat([fork, copy]), _i32([33, 33]), 33)
    assert torch.equal(read(fork), want) and torch.equal(read(copy), want)
    assert reqs.req_to_token_indexs[copy[0], :33].tolist() == remap[own].tolist() and bool((mem.mem_state[:66] == 1).all())
    q = torch.randn(2, 4, 64, generator=g).half().to(DEV)
    o, lse = lsa.longserve_fp8_decode_attention(q[:1].repeat(2, 1, 1), reqs.req_to_token_indexs, torch.cat([fork, copy]).int(), _i32([33, 33]), 33, mem.kv_buffer[1][:, :2],
                                                mem.kv_buffer[1][:, 2:], mem.kv_scales[1][:, :2], mem.kv_scales[1][:, 2:])
    assert torch.equal(o[0], o[1]) and torch.equal(lse[0], lse[1])
    reqs.free_reqs(torch.cat([fork, copy]), _i32([33, 33]), 33)
    _as_counted(mem, reqs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_prefix_over_two_instances(lsa, dtype):
    """The prefix's first tokens in one pool, its last ones and the own tokens in another: float32 partials of both, joined by lse_merge."""
    c = _case(97, 8, 2, 128, dtype, [(400, [3, 40, 0])], [])
    kv, t, r = c["kv"], c["table"], c["g"][2][0]
    want = orc.decode(c["q"], kv[:, :2], kv[:, 2:], t, c["req"], c["len"], *c["g"], 400, dtype)
    first = dict(c, table=t.clone(), len=torch.full((3,), 150, dtype=torch.int32), g=(*c["g"][:3], [150]), most=150, own=0)
    second = dict(c, table=torch.full_like(t, PAD), len=c["len"] - 150, g=(*c["g"][:3], [250]), most=250)
    second["table"][:, :-150] = t[:, 150:]
    parts = [_decode_on_gpu(lsa, x, out=torch.empty(c["q"].shape, device=DEV)) for x in (first, second)]
    o, lse = lsa.lse_merge(parts, out_dtype=dtype)
    # (each part is off by what the whole may be off by, relative to the same sums; joining adds less than the 64 eps that are counted for that)
    _check((o, lse), (want[0], want[1], 2 * want[2], 2 * want[3]), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_same_call_gives_the_same_bits(lsa, dtype):
    """Work is dealt by the sizes alone and joined in one order: repeated calls, in workspaces that hold anything, agree bit for bit."""
    c = _case(101, 32, 8, 128, dtype, [(1500, [100, 3, 700] * 6), (700, [0, 9])], [400])
    p = _prompt_case(103, 32, 8, 128, dtype, [(1200, 150), (300, 40)], tail=0)
    runs = []
    for fill in (0, 77, 255):
        ws = torch.full((lsa.shared_prefix_decode_workspace_bytes(len(c["q"]), 2, 32, 8, 128, c["most"], c["own"]),), fill, dtype=torch.uint8, device=DEV)
        pws = torch.full((lsa.shared_prefix_attention_workspace_bytes(len(p["q"]), 2, 32, 8, 128, p["most"]),), fill, dtype=torch.uint8, device=DEV)
        o, m, l = torch.zeros(p["q"].shape, dtype=dtype, device=DEV), torch.full(p["q"].shape[:2], -math.inf, device=DEV), torch.zeros(p["q"].shape[:2], device=DEV)
        _prompt_on_gpu(lsa, p, o, m, l, workspace=pws)
        runs.append((*_decode_on_gpu(lsa, c, workspace=ws), o, m, l))
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(runs[0], run))


@pytest.mark.gpu
@pytest.mark.parametrize("run", [1, 5, 90])
def test_forks_against_lists_where_slots_are_free(lsa, run):
    """Runs of forks of one source, rising and falling lengths, sources and destinations that do not exist, a quarter of the slots free."""
    g = torch.Generator().manual_seed(run)
    rows, width, size = 120, 300, 5000
    table = torch.randint(-2, size + 2, (rows, width), generator=g).int()
    state = torch.randint(0, 4, (size,), generator=g).int()
    dst = torch.randperm(100, generator=g).tolist()
    src = [100 + (i // run) % 20 for i in range(100)]
    src[7], src[50], dst[20], dst[70] = -1, rows, -3, rows + 5
    lens = torch.randint(-2, width + 20, (100,), generator=g).tolist()
    for most in (width, 170):
        want_t, want_s = orc.fork(table, src, dst, lens, most, state)
        t, st = table.to(DEV), state.to(DEV)
        lsa.fork_requests(t, _i32(src), _i32(dst), _i32(lens), most, st)
        assert torch.equal(t.cpu(), want_t) and torch.equal(st.cpu(), want_s)
