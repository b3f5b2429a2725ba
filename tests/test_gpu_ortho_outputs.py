"""GPU tests of the outputs that `orthogonalize` is given: checked where there is nothing to compute, too."""
import pytest
import torch

from laser_amd import grad_ops as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(0, 4, 5), (3, 0, 5), (4, 0), (2, 4, 5)])
def test_an_output_that_does_not_fit_is_refused(shape):
    g = torch.randn(shape, device="cuda")
    for out in (torch.empty(7, 5, dtype=torch.bfloat16, device="cuda"), torch.empty(shape, device="cuda"), torch.empty(shape, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            G.orthogonalize(g, out=out)
    out = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    assert G.orthogonalize(g, out=out) is out
