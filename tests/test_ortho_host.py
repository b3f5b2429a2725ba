"""CPU tests of the orthogonalised update's host side: workspace sizes, refusals before any launch, the parameter split."""
import ctypes as C

import pytest
import torch
from torch import nn

from laser_amd import _lib, grad_ops as G, training


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return _lib.load()


def _table(*rows):
    return (C.c_float * (3 * len(rows)))(*(v for r in rows for v in r))


NS = G.NEWTON_SCHULZ


def test_workspace_sizes(lib):
    need = lib.sgclip_orthogonalize_workspace_bytes
    assert need(0, 8, 8) == 0 and need(1, 0, 8) == 0 and need(1, 8, -1) == 0
    assert need(1, 100, 300) == need(1, 300, 100) > 0
    assert need(64, 128, 128) == 64 * need(1, 128, 128) == need(1000, 128, 128)     # larger batches run in groups
    # operands of 4 bytes an element, padded to 32 columns: X, two X^T, five squares, 64 partial sums and a factor
    assert need(1, 33, 65) == 33 * 3 * 128 + 2 * 65 * 2 * 128 + 5 * 33 * 2 * 128 + 65 * 8


def test_entry_point_refusals(lib):
    p, t5 = 4096, _table(*[NS] * 5)

    def ortho(**kw):
        a = dict(g=p, dt=0, bs=64, ld=8, batch=1, rows=8, cols=8, co=t5, steps=5, eps=1e-7, out=p, obs=64, ldo=8, ws=p, n=1 << 30)
        a.update(kw)
        return lib.sgclip_orthogonalize(*(a[k] for k in ("g", "dt", "bs", "ld", "batch", "rows", "cols", "co", "steps", "eps", "out", "obs",
                                                         "ldo", "ws", "n")), None)
    E = _lib.EINVAL
    assert ortho(batch=0) == _lib.OK
    for bad in (dict(g=None), dict(out=None), dict(dt=2), dict(ld=7), dict(ldo=7), dict(batch=-1), dict(rows=0), dict(cols=65537), dict(steps=0),
                dict(steps=33), dict(co=None), dict(eps=-1.0), dict(eps=float("nan")), dict(batch=2, obs=63)):
        assert ortho(**bad) == E, bad
        assert lib.sgclip_last_error()
    assert ortho(ws=None) == _lib.ENOSPC and ortho(n=100) == _lib.ENOSPC and ortho(ws=p + 8) == _lib.ENOSPC
    # coefficients under which singular values or a polynomial leave the range that the operands can hold
    for co in ((5000.0, 0.0, 0.0), (3.0, 0.0, 3.0), (float("nan"), 0.0, 0.0), (float("inf"), 0.0, 0.0)):
        assert ortho(co=_table(*[co] * 5)) == E, co
    one = (C.c_void_p * 1)(p)
    null = (C.c_void_p * 1)(None)

    def muon(params=one, grads=one, momenta=one, count=1, rows=8, cols=8, ws=p, n=1 << 30, co=t5, steps=5):
        return lib.sgclip_muon_step(params, grads, momenta, count, rows, cols, 0.95, 1, 1e-3, 0.0, 1.0, co, steps, 1e-7, ws, n, None)
    assert muon(count=0) == _lib.OK
    for bad in (dict(count=-1), dict(params=None), dict(grads=null), dict(momenta=null), dict(rows=0), dict(steps=0), dict(co=None)):
        assert muon(**bad) == E, bad
    assert muon(n=100) == _lib.ENOSPC


def test_python_refusals(lib):
    g = torch.randn(8, 8)
    with pytest.raises(ValueError, match="GPU"):
        G.orthogonalize(g)
    with pytest.raises(ValueError):
        G.muon_step([g], [g], [g], 1e-3)
    with pytest.raises(ValueError):
        G.muon_step([g], [], [g], 1e-3)
    G.muon_step([], [], [], 1e-3)
    with pytest.raises(ValueError, match="steps"):
        G._coefficients(NS, 0)
    with pytest.raises(ValueError, match="coefficients"):
        G._coefficients((NS, NS), 3)
    with pytest.raises(ValueError, match="coefficients"):
        G._coefficients((1.0, 2.0), 3)
    assert list(G._coefficients((NS, (1.5, -0.5, 0.0)), 2))[3:] == [1.5, -0.5, 0.0]
    with pytest.raises(ValueError, match="adjust"):
        training.Muon([nn.Parameter(g)], adjust="size")
    p = nn.Parameter(g)
    for params in ([p, p], [nn.Parameter(torch.randn(8))], [nn.Parameter(torch.randn(4, 4).double())], [nn.Parameter(torch.randn(4, 6).t())],
                   [nn.Parameter(torch.randn(0, 4))]):
        with pytest.raises(ValueError):
            training.Muon(params)


def test_groups_and_split():
    named = [("clip_cate_model.vision_model.encoder.layers.0.mlp.fc1.weight", nn.Parameter(torch.randn(8, 4))),
             ("clip_cate_model.vision_model.encoder.layers.0.mlp.fc1.bias", nn.Parameter(torch.randn(8))),
             ("clip_cate_model.vision_model.embeddings.position_embedding.weight", nn.Parameter(torch.randn(5, 4))),
             ("clip_cate_model.visual_projection.weight", nn.Parameter(torch.randn(4, 4))),
             ("clip_cate_model.text_model.encoder.layers.3.self_attn.q_proj.weight", nn.Parameter(torch.randn(4, 4))),
             ("clip_cate_model.text_model.encoder.layers.3.mlp.fc1.weight", nn.Parameter(torch.randn(8, 4)))]
    matrices, rest = training.split_for_muon(named)
    assert [tuple(p.shape) for p in matrices] == [(8, 4), (4, 4), (8, 4)] and len(rest) == 3
    opt = training.Muon(matrices)
    assert [tuple(b.shape) for b in opt.momentum] == [(2, 8, 4), (1, 4, 4)] and not any(b.any() for b in opt.momentum)
    assert opt.groups[0][1] is matrices[2]
    opt.step()                 # no gradients: nothing to do
    matrices[0].grad = torch.ones(8, 4)
    opt.zero_grad(set_to_none=False)
    assert not matrices[0].grad.any()
    opt.zero_grad()
    assert matrices[0].grad is None
