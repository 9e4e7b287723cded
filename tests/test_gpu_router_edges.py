"""The router where its numbers and its loop can go wrong: entries that another lane fills in, several rows per warp, scores far from
the largest one, logits far below zero.  Against the 64-bit form of tests/plain_forms.py."""
import itertools

import pytest
import torch

from tests import plain_forms as P
from tests.test_gpu_router import check_backward, check_forward, logits_of

pytestmark = pytest.mark.gpu

U = P.U32


@pytest.mark.parametrize("E,K", [(60, 6), (129, 7), (256, 8), (700, 32)])
@pytest.mark.parametrize("score,renorm", list(itertools.product(["softmax", "sigmoid"], [True, False])))
def test_a_warps_first_row_has_the_score_sums_gradient(score, renorm, E, K):
    """The picks' gradients are added to d_score_sums entries that other lanes have filled in: one row per warp, so that every row
    is a warp's first, and runs agree."""
    from mok import functional as F
    cfg = F.MoKRouterConfig(topk=K, score=score, renormalize=renorm)
    logits = logits_of(1500, E, torch.float32, seed=E)
    r = check_forward(cfg, logits)
    first = check_backward(cfg, logits, r)
    for _ in range(10):
        assert torch.equal(check_backward(cfg, logits, r), first)
