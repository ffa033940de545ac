"""More rows than one launch's threads can number in 32 bits."""
import pytest
import torch

import memboost_b200 as mb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [3, 8])
def test_dequantize_more_than_2_27_rows(K):
    """Rows of three values leave by the path for any alignment (a warp each),
    rows of eight by whole pieces."""
    rows = 2 ** 27 + 1003
    g = torch.Generator(device="cuda").manual_seed(K)
    codes = torch.randint(-127, 128, (rows, 16), generator=g, dtype=torch.int8,
                          device="cuda")[:, :K]
    scales = torch.rand((rows,), generator=g, device="cuda")
    got = mb.dequantize_int8(mb.Int8Tensor(codes, scales), torch.float16)
    for r0 in range(0, rows, 1 << 24):
        part = slice(r0, min(rows, r0 + (1 << 24)))
        want = (codes[part].float() * scales[part].unsqueeze(1)).half()
        assert torch.equal(got[part], want), r0
