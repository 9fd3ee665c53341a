"""The operators of an acoustic network where numbers end: outputs far from zero, non-finite adapters, the bits that sums are held in,
adapters loaded while other threads decode.  Bounds are those of tests/net_ref.py unless a test derives its own."""
import numpy as np
import pytest
import torch

import net_ref
from pocketsphinx_amd import senone_scores
from test_net_gpu import DT, _close, _dev, _layer, _off, _rand

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


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [3, 100, 1000, 6500])
def test_a_non_finite_adapter_stays_with_its_utterances(rows, dtype):
    """few rows, tiles of 128 and of 256 frames: infinities and NaN in one speaker's a or b show in that speaker's frames, in the outputs they
    feed, and nowhere else; the batch interleaves the speakers, so tiles hold several"""
    g = torch.Generator().manual_seed(620)
    d_in, d_out = 136, 5126
    layer, w, b, ad = _layer(g, DT[dtype], d_in, d_out, [16, 3, 20, 16], 40)
    lens = [1, rows // 5, 0, 1, rows // 3, 1]
    lens += [1] * min(rows, 40)
    lens += [max(0, rows - sum(lens))]
    slots = [(2 * u + 1) % 5 - 1 for u in range(len(lens))]             # -1 .. 3
    off = _off(lens)
    x = _rand(g, off[-1], d_in, dtype=DT[dtype])
    want, err = net_ref.proj(x, w, b, ad, off, slots)
    row_slot = torch.tensor([slots[u] for u, n in enumerate(lens) for _ in range(n)])
    inf, nan = float("inf"), float("nan")
    a1, b1, s1 = ad[1]
    b1 = b1.clone()
    b1[7, 1], b1[2500, 2], b1[d_out - 1, 0] = inf, nan, -inf
    layer.set_adapter(1, a1, b1, s1)
    a2, b2, s2 = ad[2]
    a2 = a2.clone()
    a2[19, d_in - 1], a2[0, 3] = inf, nan
    layer.set_adapter(2, a2, b2, s2)
    for out_dtype in {DT[dtype], torch.float32}:
        got = layer(x.cuda(), _dev(off), _dev(slots), out_dtype=out_dtype).double().cpu()
        other = (row_slot != 1) & (row_slot != 2)
        _close(got[other], want[other], err[other], out_dtype, "other speakers")
        hit = torch.zeros(d_out, dtype=torch.bool)
        hit[[7, 2500, d_out - 1]] = True
        one = got[row_slot == 1]
        assert not torch.isfinite(one[:, hit]).any()
        _close(one[:, ~hit], want[row_slot == 1][:, ~hit], err[row_slot == 1][:, ~hit], out_dtype, "the outputs that the infinity does not feed")
        assert not torch.isfinite(got[row_slot == 2]).any()
