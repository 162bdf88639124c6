"""GPU: refusals of the MXFP4 products that need a device to be reached; each is a ValueError."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_bias_without_dimensions():
    from flash_mh_moe.mxfp4 import MXFP4Matrix, mxfp4_expert_linear, mxfp4_linear
    w = MXFP4Matrix.from_blocks(torch.zeros(1, 16, dtype=torch.uint8, device="cuda"),
                                torch.full((1, 1), 127, dtype=torch.uint8, device="cuda"))
    w3 = MXFP4Matrix.from_blocks(*(t[None] for t in w.to_blocks()))
    x = torch.ones(3, 32, device="cuda")
    offs = torch.tensor([0, 3], device="cuda")
    for b in (torch.tensor(1.0, device="cuda"), torch.ones(2, device="cuda"), torch.ones(1, 2, device="cuda")):
        with pytest.raises(ValueError, match="bias"):
            mxfp4_linear(x, w, b)
        with pytest.raises(ValueError, match="bias"):
            mxfp4_expert_linear(x, w3, offs, bias=b)
    assert (mxfp4_linear(x, w, torch.ones(1, device="cuda")) == 1).all()
    assert (mxfp4_expert_linear(x, w3, offs, bias=torch.ones(1, 1, device="cuda")) == 1).all()
