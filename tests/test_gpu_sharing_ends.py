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
