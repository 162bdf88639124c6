"""CPU: MXFP4 matrices and arguments at the edges of their shapes."""
import pytest
import torch


@pytest.mark.parametrize("n,rows,cols", [(0, 4, 32), (0, 0, 7), (2, 0, 32), (0, 130, 300)])
def test_blocks_of_nothing(n, rows, cols):
    from flash_mh_moe.mxfp4 import MXFP4Matrix
    d = torch.zeros(n, rows, (cols + 1) // 2, dtype=torch.uint8)
    s = torch.zeros(n, rows, (cols + 31) // 32, dtype=torch.uint8)
    m = MXFP4Matrix.from_blocks(d, s, cols)
    assert m.shape == (n, rows, cols)
    d2, s2 = m.to_blocks()
    assert d2.shape == d.shape and s2.shape == s.shape
