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


@pytest.mark.gpu
@pytest.mark.parametrize("own", [1, 100, 200, 2000])
def test_decode_steps_in_one_workspace(lsa, own):
    """Close bounds of the own tokens, from the first step to the last, in the workspace of the longest."""
    ws = torch.empty(lsa.shared_prefix_decode_workspace_bytes(64, 1, 32, 8, 128, 4000, 3000), dtype=torch.uint8, device=DEV)
    c = _case(51, 32, 8, 128, torch.float16, [(4000, [own] * 40)], [])
    got, want = _decode_on_gpu(lsa, c, workspace=ws), _decode_on_gpu(lsa, c)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
