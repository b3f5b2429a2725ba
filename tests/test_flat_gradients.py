"""CPU tests of gradients that live in a `FlatParameters` buffer: every way of clearing them leaves `.grad` the buffer's views, and
nothing in the buffer that no `.grad` shows."""
import gc
import types

import pytest
import torch
from torch import nn

from laser_amd import training


def flattened():
    named = [("m.encoder.layers.0.fc1.weight", nn.Parameter(torch.randn(8, 4))), ("m.encoder.layers.0.fc1.bias", nn.Parameter(torch.randn(7))),
             ("m.encoder.layers.0.fc2.weight", nn.Parameter(torch.randn(4, 8))), ("m.logit_scale", nn.Parameter(torch.tensor(1.0)))]
    flat = training.FlatParameters(named)
    flat.grad.copy_(torch.randn(flat.total))
    return named, flat


def is_place(flat, name, p):
    return p.grad is not None and p.grad.shape == p.shape and p.grad.data_ptr() == flat.grad.data_ptr() + 4 * flat.index[name][0]


@pytest.mark.parametrize("set_to_none", [True, False])
def test_zero_grad_of_optimisers_of_single_parameters(set_to_none):
    named, flat = flattened()
    matrices, rest = training.split_for_muon(named)
    for opt in (training.Muon(matrices), training.Adam(rest)):
        opt.zero_grad(set_to_none=set_to_none)
    assert all(is_place(flat, n, p) for n, p in named)
    assert all(not flat.grad_view(n).any() for n, _ in named)
    flat.grad_view("m.encoder.layers.0.fc2.weight").add_(3.0)        # what a tower's backward does
    assert (matrices[1].grad == 3.0).all()


def test_zero_grad_takes_back_a_dropped_view():
    named, flat = flattened()
    for _, p in named:
        p.grad = None
    for opt in (training.Muon([named[0][1], named[2][1]]), training.Adam([named[1][1], named[3][1]])):
        opt.zero_grad()
    assert all(is_place(flat, n, p) and not p.grad.any() for n, p in named)


def test_other_parameters_as_before():
    p, q = nn.Parameter(torch.randn(3, 4)), nn.Parameter(torch.randn(3, 4))
    for opt in (training.Muon([p, q]), training.Adam([p, q])):
        p.grad = torch.ones(3, 4)
        opt.zero_grad(set_to_none=False)
        assert not p.grad.any() and q.grad is None
        opt.zero_grad()
        assert p.grad is None
    named, flat = flattened()
    del flat
    gc.collect()
    opt = training.Adam([p for _, p in named])
    opt.zero_grad()          # the buffer's owner is gone, and with it whoever would add to it
    assert all(p.grad is None for _, p in named)


def test_a_tower_starts_from_zeros_where_the_view_was_dropped():
    named, flat = flattened()
    kept = named[1][1].grad.clone()
    named[0][1].grad = named[2][1].grad = None       # torch's own zero_grad on some of them
    sink = training.GradSink(types.SimpleNamespace(flat=flat, flat_prefix="m."))
    sink.get("encoder.layers.0.fc1.weight").add_(2.0)
    assert (named[0][1].grad == 2.0).all() and not named[2][1].grad.any() and torch.equal(named[1][1].grad, kept)
    assert all(is_place(flat, n, p) for n, p in named)
    sink = training.GradSink(types.SimpleNamespace(flat=flat, flat_prefix="m."))     # the next chunk's or batch's adds to them
    sink.get("encoder.layers.0.fc1.weight").add_(2.0)
    assert (named[0][1].grad == 4.0).all()


def test_a_reduced_step_starts_with_every_view_in_place():
    named, flat = flattened()
    reducer = training.GradientReducer(flat, [("all", 0, flat.total)])
    for _, p in named:
        p.grad = None
    reducer.begin()
    assert all(is_place(flat, n, p) and not p.grad.any() for n, p in named)
    (named[3][1] * 5).backward()                     # a parameter whose gradient autograd adds
    assert flat.grad_view("m.logit_scale").item() == 5.0


def test_a_gradient_beside_the_buffer_moves_into_it():
    """torch's zero_grad, then a backward pass: autograd gives a parameter outside the towers a tensor of its own."""
    named, flat = flattened()
    scale = named[3][1]
    for _, p in named:
        p.grad = None
    (scale * 5).backward()
    assert not is_place(flat, "m.logit_scale", scale)
    training.GradSink(types.SimpleNamespace(flat=flat, flat_prefix="m."))
    assert all(is_place(flat, n, p) for n, p in named)
    assert scale.grad.item() == 5.0 and not named[0][1].grad.any()
    (scale * 2).backward()
    assert flat.grad_view("m.logit_scale").item() == 7.0


def test_flat_adam_reads_every_gradient(monkeypatch):
    named, flat = flattened()
    opt = training.Adam(flat)
    seen = []
    monkeypatch.setattr(training.G, "adamw", lambda p, g, *a: seen.append(g.clone()))
    for _, p in named:
        p.grad = None
    (named[3][1] * 5).backward()
    opt.step()
    for n, (at, count, _) in flat.index.items():       # what lies between them, for alignment, is no parameter's
        assert seen[0][at:at + count].sum().item() == (5.0 if n == "m.logit_scale" else 0.0)


def test_flat_zero_grad_clears_what_lies_beside_the_buffer():
    named, flat = flattened()
    for _, p in named:
        p.grad = None
    (named[3][1] * 5).backward()
    flat.zero_grad()
    assert all(is_place(flat, n, p) and not p.grad.any() for n, p in named)
    (named[3][1] * 2).backward()
    flat.attach_gradients()
    assert named[3][1].grad.item() == 2.0
