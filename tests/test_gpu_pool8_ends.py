"""Decode over the 8-bit pool where its exponents are at their ends: slots that nobody wrote, V rows of zeros, very small and very large ones."""
import pytest
import torch

from tests.test_gpu_pool8 import Case

K8 = ["e4m3-f16", "e4m3-bf16"]


class Unwritten(Case):
    """A Case whose slots that no request holds, slot 0 among them, have the exponent byte 255 (E8M0's NaN) beside their NaN rows."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        n = self.values.shape[0]
        used = torch.zeros(n, dtype=torch.bool)
        used[self.table[(self.table >= 0) & (self.table < n)].long()] = True
        if used[0]:
            to = int((~used).nonzero()[0])
            self.table[self.table == 0] = to
            used[0], used[to] = False, True
            for t in (self.values, self.pool.view(torch.uint8), self.scales):
                t[[0, to]] = t[[to, 0]]
        self.scales[(~used).cuda()] = 255
        assert not used[0] and not (self.table == 0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", K8)
@pytest.mark.parametrize("lens,holes", [([1, 33, 700, 0, 64], []), ([70, 40], [(0, 0), (0, 33), (0, 34), (1, 39)]),
                                        ([9000, 3], [(0, 0), (0, 8999), (0, 4000), (1, 1)]), ([96, 96, 96], [])])
def test_exponents_of_slots_that_are_not_seen_do_not_matter(lsa, kind, lens, holes):
    """Slots are neutral where a position does not exist (past a request's end, a hole of the table), whatever slot 0 holds; in both launch forms."""
    c = Unwritten(kind, len(lens), 8, 2, 128, lens, seed=21, holes=holes)
    for max_len in (None, 1 << 17):
        c.check(c.run(lsa, max_len=max_len))
        c.check(c.run(lsa, 50, 3, max_len=max_len), 50, 3)
