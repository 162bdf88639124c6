"""GPU: mxfp4_expert_linear's ``out`` as autograd sees it: a tensor that is written in place."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs():
    from flash_mh_moe.mxfp4 import MXFP4Matrix
    g = torch.Generator(device="cuda").manual_seed(0)
    w = MXFP4Matrix.from_blocks(torch.randint(0, 256, (2, 64, 32), generator=g, device="cuda", dtype=torch.uint8),
                                torch.randint(118, 126, (2, 64, 2), generator=g, device="cuda", dtype=torch.uint8))
    return torch.randn(6, 64, generator=g, device="cuda"), w, torch.tensor([0, 2, 5], device="cuda")


def test_out_counts_as_changed():
    from flash_mh_moe.mxfp4 import mxfp4_expert_linear
    x, w, offs = _inputs()
    buf = torch.zeros(6, 70, device="cuda")
    v = buf._version
    mxfp4_expert_linear(x, w, offs, out=buf[:, :64])
    assert buf._version > v
    # what autograd saved of it before is refused, not used with other values
    a = torch.ones(6, 64, device="cuda", requires_grad=True)
    out = torch.ones(6, 64, device="cuda")
    y = (a * out).sum()
    mxfp4_expert_linear(x, w, offs, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_out_that_needs_a_gradient_is_refused():
    from flash_mh_moe.mxfp4 import mxfp4_expert_linear
    x, w, offs = _inputs()
    out = torch.zeros(6, 64, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="backward"):
        mxfp4_expert_linear(x, w, offs, out=out)
    with torch.no_grad():
        assert mxfp4_expert_linear(x, w, offs, out=out) is out
    with torch.inference_mode():
        buf = torch.zeros(6, 64, device="cuda")
        assert torch.equal(mxfp4_expert_linear(x, w, offs, out=buf), out)
