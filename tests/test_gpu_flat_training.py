"""GPU tests of the documented train loop of a flattened model with an optimiser for its matrices and one for the rest."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from laser_amd import training  # noqa: E402
from laser_amd.synthetic import make_clip_batch  # noqa: E402
from test_gpu_train import _loss, _setup  # noqa: E402


def _model():
    b = make_clip_batch(17, n_videos=1, frames=2, objects=3, H=96, W=128, k_cate=4, k_unary=5, k_binary=3, min_box=12, max_box=90)
    model = _setup(31, float(np.log(10.0)))[3].enable_training()
    return model, b.forward_kwargs()


def _near(a, b):
    """Two backward passes of one loss: atomics in another order."""
    return ((a - b).norm() / b.norm()).item() <= 1e-4


def test_documented_loop():
    model, kw = _model()
    reducer = model.gradient_reducer()               # flattens
    flat = model.flatten_parameters()
    matrices, rest = training.split_for_muon(model.named_parameters())
    opts = training.Muon(matrices, lr=2e-4), training.Adam(rest, lr=1e-5)
    for _ in range(3):
        for o in opts:
            o.zero_grad()
        reducer.begin()
        _loss(model(**kw), 4)[0].backward()
        reducer.finish()
        got = flat.grad.clone()
        assert all(p.grad is not None and torch.equal(p.grad, flat.grad_view(n)) for n, p in model.named_parameters())
        flat.zero_grad()
        _loss(model(**kw), 4)[0].backward()
        assert _near(got, flat.grad)
        before = [p.detach().clone() for p in matrices]
        for o in opts:
            o.step()
        assert all(not torch.equal(p, q) for p, q in zip(matrices, before))
    torch.cuda.synchronize()


def test_gradients_dropped_by_the_module_itself():
    model, kw = _model()
    flat = model.flatten_parameters()
    _loss(model(**kw), 4)[0].backward()
    towers = [n for n in flat.index if not n.endswith("logit_scale")]
    once = torch.cat([flat.grad_view(n).reshape(-1) for n in towers])
    model.zero_grad(set_to_none=True)
    _loss(model(**kw), 4)[0].backward()
    again = torch.cat([flat.grad_view(n).reshape(-1) for n in towers])
    assert _near(again, once)
    named = dict(model.named_parameters())
    assert all(torch.equal(named[n].grad, flat.grad_view(n)) for n in towers)
    torch.cuda.synchronize()
