"""GPU tests of the orthogonalised updates' precision where a few directions dominate the others: what is lost there is lost in the
Gram matrix, whose small eigenvalues the iteration raises most.

Tolerance, absolute in the Frobenius norm, with |X| = 1 at the start and roundings of u = 2^-23 (an operand of 22 bits):
  the roundings of X and of what is applied to it grow by a per step that remains: four in each of five steps, 20 a^5 u;
  in a block of two steps on one Gram matrix A a rounding E of it, |E|_F <= u, reaches the second step's Gram matrix as a^2 E: the
  product of the block's polynomials is off by at most a (|b| + 2 |c|) (1 + a^2) |E|_2.  The roundings of A's elements are apart from
  each other, which leaves E a spectral norm of at most 2.5 / sqrt(m) of its Frobenius norm, 0.16 for m >= 256, the shortest side with
  such blocks.  Three blocks in five steps: 3 (|b| + 2 |c|) (1 + a^2) / a 0.16 = 16 a^5 u.
Together 36 a^5 u = 2.1e-3 (and 20 a^5 u where every step has a Gram matrix of its own), whatever |O| is."""
import pytest
import torch

from laser_amd import grad_ops as G
from test_gpu_ortho import BF16, F64, UBF, iterate, raw, rel

pytestmark = pytest.mark.gpu

A5U = G.NEWTON_SCHULZ[0] ** 5 * 2.0 ** -23


def of_singular_values(s, rows, cols):
    m = len(s)
    u = torch.linalg.qr(torch.randn(rows, m, dtype=F64))[0]
    v = torch.linalg.qr(torch.randn(cols, m, dtype=F64))[0]
    return ((u * s) @ v.t()).float().cuda()


def matrix(kind, rows, cols):
    m = min(rows, cols)
    noise = torch.randn(rows, cols, device="cuda")
    if kind == "mean":
        return 1 + 0.02 * noise
    if kind == "mean and little noise":
        return 1 + 0.003 * noise
    if kind == "same rows":
        g = 0.003 * noise
        g[:4] += torch.randn(cols, device="cuda")
        return g
    if kind == "steps":          # groups of rows, each constant
        return 2.0 ** (torch.arange(rows, device="cuda") * 4 // rows).float()[:, None] + 0.01 * noise
    i = torch.arange(m, dtype=F64)
    if kind == "power law":
        return of_singular_values(1 / (1 + i), rows, cols)
    return of_singular_values(torch.where(i < 1, 1.0, 1e-3), rows, cols)


KINDS = ["mean", "mean and little noise", "same rows", "steps", "power law", "one direction"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(256, 1024), (320, 400), (768, 1536), (2048, 512), (1000, 257)])
def test_dominated_matrices(rows, cols, kind):
    torch.manual_seed(rows + cols)
    g = matrix(kind, rows, cols)
    want = iterate(g)
    assert (raw(g).double() - want).norm() <= 36 * A5U
    assert (G.orthogonalize(g).double() - want).norm() <= 36 * A5U + UBF * want.norm()
    b = g.to(BF16)
    want = iterate(b)
    assert (G.orthogonalize(b).double() - want).norm() <= 36 * A5U + UBF * want.norm()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(100, 90), (128, 256), (60, 1000), (300, 300), (200, 700)])
def test_dominated_matrices_step_by_step(rows, cols, kind):
    torch.manual_seed(rows + cols)
    g = matrix(kind, rows, cols)
    want = iterate(g)
    assert (raw(g).double() - want).norm() <= 20 * A5U


@pytest.mark.parametrize("rows,cols", [(96, 100), (90, 700), (300, 310), (300, 900), (900, 300)])
def test_converging_iteration_ends_orthonormal(rows, cols):
    """Singular values from 0.2 to 1 of the largest are at least 0.2 / sqrt(300) = 0.0115 of the norm; s (3 - s^2) / 2 brings that to 0.42
    in nine steps and to 1 - 1e-9 in six more.  From there a step's errors do not grow (the derivative at 1 is none), and what the
    last one leaves is its roundings of 22 bits and its sums over up to 900 products in fp32, 30 roundings of 2^-24 each: below 1e-5."""
    torch.manual_seed(rows)
    m = min(rows, cols)
    g = of_singular_values(torch.linspace(0.2, 1.0, m, dtype=F64), rows, cols)
    o = raw(g, steps=18, coefficients=(1.5, -0.5, 0.0)).double()
    o = o if rows <= cols else o.t()
    gram = o @ o.t().contiguous()
    # 22 bits per operand of the last step, and its sums
    assert (gram - torch.eye(m, device="cuda", dtype=F64)).abs().max() <= 1e-5
    assert rel(o if rows <= cols else o.t(), iterate(g, 18, (1.5, -0.5, 0.0))) <= 1e-5
