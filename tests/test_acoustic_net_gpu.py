"""The operators of an acoustic network where numbers end: outputs far from zero, non-finite adapters, the bits that sums are held in,
adapters loaded while other threads decode.  Bounds are those of tests/net_ref.py unless a test derives its own."""
import numpy as np
import pytest
import torch

import net_ref
from pocketsphinx_amd import senone_scores
from test_net_gpu import DT, _rand

pytestmark = pytest.mark.gpu


def _best_of(z, prior):
    """(best, bound): max(z - prior) - log sum exp z with the row's greatest taken off first, in 64 bits.  The bound is net_ref.senones's and
    two roundings of numbers as large as the greatest in 64 bits (z - prior, the logarithm), 2^-53 of it each."""
    z, p = z.double().cpu().numpy(), prior.double().cpu().numpy()
    m = z.max(axis=1)
    with np.errstate(invalid="ignore"):
        best = ((z - m[:, None]) - p).max(axis=1) - np.log(np.exp(z - m[:, None]).sum(axis=1))
    return best, (z.shape[1] + 110) * 2 * net_ref.U + np.abs(best) * net_ref.U + np.abs(m) * 2.0 ** -52


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows, n_sen", [(24, 3), (24, 100), (24, 5126), (600, 5126), (24, 25000), (24, 45000)])
def test_best_of_outputs_far_from_zero(rows, n_sen, dtype):
    """rows whose greatest output is far from zero: all alike, some masked, one above the others, spread about it; rows of the other kind
    between them are as ever"""
    g = torch.Generator().manual_seed(600 + n_sen)
    z = _rand(g, rows, n_sen, dtype=DT[dtype], scale=4.0)
    r = 0
    for far in (-1e10, 1e10, 1e20, -1e30, -3e37, 3e38, -1e6, 3e9):
        z[r] = far
        z[r + 1] = far
        z[r + 1, 1::2] = -float("inf")
        z[r + 2] = (far + z[r + 2].double()).to(DT[dtype])
        r += 3
    prior = torch.log_softmax(_rand(g, n_sen).double(), 0).float()
    want, err = _best_of(z, prior)
    for dp, w, e in ((prior.cuda(), want, err), (None,) + _best_of(z, torch.zeros(n_sen))):
        _, b = senone_scores(z.cuda(), dp, scale=0.8, want_best=True)
        b = b.double().cpu().numpy()
        bad = ~(np.abs(b - w) <= e)
        assert not bad.any(), "rows %r: %r, not %r +- %r" % (np.nonzero(bad)[0].tolist(), b[bad], w[bad], e[bad])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_sen", [2, 100, 5126, 45000])
def test_best_of_every_non_finite_row(n_sen, dtype):
    """nothing but masked senones: -inf; a NaN or an output of +inf (inf - inf): NaN, and no other row's"""
    g = torch.Generator().manual_seed(610 + n_sen)
    z = _rand(g, 9, n_sen, dtype=DT[dtype], scale=4.0)
    inf = float("inf")
    z[0] = -inf
    z[2, n_sen // 2] = float("nan")
    z[3] = float("nan")
    z[5, n_sen - 1] = inf
    z[6] = inf
    z[7] = -inf
    z[7, 0] = float("nan")
    s, b = senone_scores(z.cuda(), None, want_best=True)
    b = b.double().cpu()
    assert b[0] == -inf and torch.isnan(b[[2, 3, 5, 6, 7]]).all()
    ws, wb, be = net_ref.senones(z, None, 1.0, 1.0001)
    assert np.array_equal(s.cpu().numpy(), ws)
    for r in (1, 4, 8):
        assert abs(float(b[r]) - wb[r]) <= be[r]
