"""CPU: operators without a forward-mode derivative refuse dual tensors; a result without its tangent would
look like one whose derivative is zero.  The refusal comes before the device is looked at."""
import pytest
import torch
import torch.autograd.forward_ad as fwad


def _w(n=None):
    from flash_mh_moe.mxfp4 import MXFP4Matrix
    lead = (4,) if n is None else (n, 4)
    return MXFP4Matrix.from_blocks(torch.zeros(*lead, 16, dtype=torch.uint8), torch.zeros(*lead, 1, dtype=torch.uint8))


def _calls():
    from flash_mh_moe.mxfp4 import mxfp4_expert_linear, mxfp4_linear
    from flash_mh_moe.route import route_experts
    x, r = torch.zeros(3, 32), torch.ones(3)
    offs = torch.tensor([0, 1, 3])
    return {
        "route_experts": (lambda t: route_experts(t, 2), torch.zeros(1, 2, 8)),
        "linear x": (lambda t: mxfp4_linear(t, _w()), x),
        "linear bias": (lambda t: mxfp4_linear(x, _w(), t), torch.zeros(4)),
        "experts x": (lambda t: mxfp4_expert_linear(t, _w(2), offs), x),
        "experts weights": (lambda t: mxfp4_expert_linear(x, _w(2), offs, row_weights=t), r),
        "experts bias": (lambda t: mxfp4_expert_linear(x, _w(2), offs, bias=t), torch.zeros(2, 4)),
        "experts out": (lambda t: mxfp4_expert_linear(x, _w(2), offs, out=t), torch.zeros(3, 4)),
    }


@pytest.mark.parametrize("name", ["route_experts", "linear x", "linear bias", "experts x", "experts weights", "experts bias",
                                  "experts out"])
@pytest.mark.parametrize("grad", [True, False])
def test_dual_tensors_are_refused(name, grad):
    call, primal = _calls()[name]
    with torch.set_grad_enabled(grad), fwad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            call(fwad.make_dual(primal, torch.ones_like(primal)))
        with pytest.raises(ValueError, match="CUDA"):              # a tensor without a tangent goes on as before
            call(primal)
