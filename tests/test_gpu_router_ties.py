"""Which experts the router takes where many logits are equal, over all of its lane layouts and numbers of slots: the
choice is exact, so whole numbers have to be equal to the definition's. With 129 experts or more and 4 to 8 slots the
choice is among candidates, those from the smallest of eight eighths' maxima on, 64 at most; the tokens here have
few of them, about 32, and more than 64, and equal ones among the last taken and the first left.
"""
import math

import pytest

from test_gpu_router import Forward, check_forward, reference

pytestmark = pytest.mark.gpu
EXPERTS = [8, 40, 70, 128, 129, 200, 256, 300, 512, 777, 1024]


@pytest.mark.parametrize("k", [1, 4, 6, 8, 9, 16])
@pytest.mark.parametrize("e", EXPERTS)
def test_whole_numbered_logits(cuda, e, k):
    """Few levels (most slots tie), many levels, all equal, zeros of both signs, experts closed."""
    import torch
    g = torch.Generator(device=cuda).manual_seed(e + k)
    draw = lambda hi, t: torch.randint(0, hi, (t, e), device=cuda, generator=g).float()  # noqa: E731
    zeros = torch.zeros(6, e, device=cuda)
    zeros[:, 1::2] = -0.0
    zeros[3:, ::5] = 1.0
    closed = draw(4, 12)
    closed[:, torch.rand(e, device=cuda, generator=g) < 0.7] = -math.inf
    closed[:4, 2:] = -math.inf
    logits = torch.cat([draw(2, 12), draw(5, 12), draw(60, 12), draw(1000, 12), draw(1, 4) + 3.0, draw(1, 4) - 7.0, zeros, closed])
    fw = Forward(logits, k)
    check_forward(fw, reference(logits, k, True, None))


@pytest.mark.parametrize("distinct", [False, True], ids=["equal", "distinct"])
@pytest.mark.parametrize("count", [8, 9, 31, 32, 33, 40, 63, 64, 65, 100])
@pytest.mark.parametrize("e,k", [(256, 4), (256, 8), (250, 7), (512, 5), (500, 8), (1024, 8)])
def test_counts_of_candidates(cuda, e, k, count, distinct):
    """Exactly `count` experts at or above the smallest of the eighths' maxima: 1 in the first expert of each eighth,
    the others anywhere, all of them 1 or (but for the first eighth's) above."""
    import torch
    lane = 8 if e <= 256 else 16 if e <= 512 else 32
    g = torch.Generator().manual_seed(count + e)
    rows = []
    for _ in range(24):
        row = -1.0 - torch.rand(e, generator=g)
        firsts = list(range(0, e, 4 * lane))
        assert len(firsts) == 8
        rest = [x for x in torch.randperm(e, generator=g).tolist() if x not in firsts][:count - 8]
        taken = torch.tensor(firsts + rest)
        row[taken] = 1.0
        if distinct:
            above = taken[taken >= 4 * lane]
            row[above] = 1.0 + torch.randperm(len(above), generator=g).float() / 64
        rows.append(row)
    logits = torch.stack(rows).to(cuda)
    fw = Forward(logits, k)
    check_forward(fw, reference(logits, k, True, None))
