"""The block-scaled and grouped products where their inputs leave the ordinary range, on every tile form
that the sizes choose: gates far below zero, scales whose product leaves FP32, non-finite values and
partial boxes on pairs of SMs, streams that join, a quantiser past 2^31 elements."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import tsfm_b200 as tb  # noqa: E402
from test_linear_blocks_gpu import CODE, E4M3, Case, gen, ptr, quantize, stream, up  # noqa: E402

pytestmark = pytest.mark.gpu

@pytest.mark.parametrize("M,N,K", [(8000, 1000, 768), (9001, 1001, 392), (7000, 1300, 768)])
def test_partial_boxes_leave_the_padding(M, N, K):
    # 16-bit outputs of 256 x 256 tiles leave in boxes of 64 columns x 32 rows: the last ones are clipped to
    # N columns (odd ones too) and M rows, the padding of a row is left as it was
    assert N % 64
    c = Case(M, N, K, "e4m3", bias=True, seed=24)
    for dtype in (torch.bfloat16, torch.float16):
        c.check(dtype, pad=-N % 8)
        c.check(dtype, act=1, pad=-N % 8 + 24)
        c.check(dtype, pad=-N % 8 + 8, shift=8)
    g = Case(M, N, K, "e4m3", counts=[M // 2, 0, 3, M - M // 2 - 10], first=4, bias=True, seed=25)
    g.check(torch.bfloat16, pad=-N % 8 + 24)
