"""The operators of an acoustic network where numbers end: outputs far from zero, non-finite adapters, the bits that sums are held in,
adapters loaded while other threads decode.  Bounds are those of tests/net_ref.py unless a test derives its own."""
import threading

import numpy as np
import pytest
import torch

import net_ref
from pocketsphinx_amd import AdaptedProjection, group_norm, senone_scores
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


def _as_32_bits(got, want, terms, what):
    """the root mean square of the error against that of the values.  A sum of n products of like size kept in 32 bits: after i of them the
    sum is about sqrt(i) of one, and adding the next rounds it by at most U, U / sqrt 3 in the mean square; the n errors add up to
    U n / sqrt 6 of one product, U sqrt(n / 6) of the sum.  `terms`: of the sums that feed one another, one after another; the store to 32 bits
    is U / sqrt 3."""
    rel = float(((got.double() - want) ** 2).mean().sqrt() / (want ** 2).mean().sqrt())
    assert rel <= net_ref.U * (sum(terms) / 6 + 1 / 3) ** 0.5, "%s: off by %.3g, %.3g is 32 bits' due" % (what, rel, net_ref.U * (sum(terms) / 6 + 1 / 3) ** 0.5)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows, d_in, d_out", [(3, 1024, 1024), (40, 1024, 1024), (1000, 256, 5126), (6500, 256, 5126), (6500, 1024, 5126)])
def test_sums_keep_32_bits(rows, d_in, d_out, dtype):
    """into float32: the shared product, the adapter's alone, of one adapter for all frames and of several in a tile"""
    g = torch.Generator().manual_seed(630)
    w = _rand(g, d_out, d_in, dtype=DT[dtype], scale=d_in ** -0.5)
    ad = [(_rand(g, 32, d_in, dtype=DT[dtype], scale=d_in ** -0.5), _rand(g, d_out, 32, dtype=DT[dtype])) for _ in range(2)]
    x = _rand(g, rows, d_in, dtype=DT[dtype]).cuda()
    xd = x.double()
    _as_32_bits(AdaptedProjection(w)(x, out_dtype=torch.float32), xd @ w.cuda().double().t(), [d_in], "the shared product")
    alone = AdaptedProjection(torch.zeros_like(w), None, 2, 32)
    term = []
    for k, (a, b) in enumerate(ad):
        alone.set_adapter(k, a, b)
        term.append((xd @ a.cuda().double().t()) @ b.cuda().double().t())
    _as_32_bits(alone(x, _dev([0, rows]), _dev([1]), out_dtype=torch.float32), term[1], [d_in, 5 * 32], "one adapter")
    slots = torch.arange(rows) % 2
    want = torch.where(slots.cuda()[:, None] == 0, term[0], term[1])
    _as_32_bits(alone(x, _dev(list(range(rows + 1))), _dev(slots.tolist()), out_dtype=torch.float32), want, [d_in, 5 * 32], "two adapters")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_a_frames_answer_hardly_hangs_on_its_batch(dtype):
    """the same frames among two, few, many of their own speaker and many of others: sums in another order, each in 32 bits"""
    g = torch.Generator().manual_seed(640)
    d_in, d_out = 512, 5126
    layer = AdaptedProjection(torch.zeros(d_out, d_in, dtype=DT[dtype]), None, 2, 24)
    for k in range(2):
        layer.set_adapter(k, _rand(g, 24, d_in, dtype=DT[dtype], scale=d_in ** -0.5), _rand(g, d_out, 24, dtype=DT[dtype]))
    x = _rand(g, 6500, d_in, dtype=DT[dtype]).cuda()
    first = layer(x[:2], _dev([0, 2]), _dev([1]), out_dtype=torch.float32).double()
    for n in (40, 1000, 6500):
        _as_32_bits(layer(x[:n], _dev([0, n]), _dev([1]), out_dtype=torch.float32)[:2], first, [2 * d_in, 2 * 5 * 24], "%d frames" % n)
        _as_32_bits(layer(x[:n], _dev([0, 2, n]), _dev([1, 0]), out_dtype=torch.float32)[:2], first, [2 * d_in, 2 * 5 * 24], "%d frames of two" % n)


@pytest.mark.parametrize("rows", [2, 40, 1000, 6500])
def test_an_infinite_input_of_float16(rows):
    """an infinity in x goes through a (of one rank) and b as the formula says; b's values have a second part of 0 here"""
    g = torch.Generator().manual_seed(650)
    d_in, d_out, r = 136, 5126, 32
    layer = AdaptedProjection(torch.zeros(d_out, d_in, dtype=torch.float16), None, 1, r)
    a, b = _rand(g, r, d_in, dtype=torch.float16).abs() + 1, torch.sign(_rand(g, d_out, 1, dtype=torch.float16)).expand(d_out, r).contiguous()
    layer.set_adapter(0, a, b)
    x = torch.zeros(rows, d_in, dtype=torch.float16)
    x[:, 2] = 1.0
    x[rows - 1, 2] = float("inf")
    y = layer(x.cuda(), _dev([0, rows]), _dev([0])).cpu()
    # (W is 0 and meets the infinity: the shared product alone makes NaN of that row)
    assert torch.isnan(y[rows - 1]).all() and torch.isfinite(y[:rows - 1]).all()
    layer = AdaptedProjection(torch.ones(d_out, 1, dtype=torch.float16).mul_(b[:, :1]).expand(d_out, d_in).contiguous(), None, 1, r)
    layer.set_adapter(0, a, b)
    x[rows - 1] = 1.0
    x[rows - 1, 2] = float("inf")
    y = layer(x.cuda(), _dev([0, rows]), _dev([0])).cpu()
    assert torch.equal(y[rows - 1].float(), b[:, 0].float() * float("inf"))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rank", [1, 5, 33])
@pytest.mark.parametrize("rows, d_out", [(3, 330), (40, 330), (1000, 5126), (6500, 5126), (20000, 60)])
def test_non_finite_inputs_go_through_as_the_formula_says(rows, d_out, rank, dtype):
    """rows of one speaker and of two in turn with an infinity or a NaN in x: every output as in 64 bits, non-finite ones alike"""
    g = torch.Generator().manual_seed(660 + rank)
    d_in = 75
    w = _rand(g, d_out, d_in, dtype=DT[dtype])
    layer = AdaptedProjection(w, None, 2, 40)
    ad = {}
    for k in range(2):          # one sign in a row of b and in a: an infinity's terms do not meet one of the other sign among the ranks
        ad[k] = (_rand(g, rank, d_in, dtype=DT[dtype]).abs() + 0.5, (torch.sign(_rand(g, d_out, 1)) * (_rand(g, d_out, rank).abs() + 0.5)).to(DT[dtype]), 0.5)
        layer.set_adapter(k, *ad[k])
    x = _rand(g, rows, d_in, dtype=DT[dtype])
    inf = float("inf")
    x[0, d_in - 1], x[rows // 2, 3], x[rows - 1, 0] = inf, float("nan"), -inf
    for off, slots in (([0, rows], [1]), (_off([1] * rows), [t % 2 for t in range(rows)])):
        want, err = net_ref.proj(x, w, None, ad, off, slots)
        got = layer(x.cuda(), _dev(off), _dev(slots))
        _close(got, want, err, DT[dtype], "finite outputs")
        got = got.double().cpu()
        assert torch.isinf(want).sum() > d_out // 2
        assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN"
        assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]), "infinities"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_adapters_loaded_by_several_threads(dtype):
    """two threads load their speakers from the host, over and over, while two others decode on streams of their own: every output is that of
    one whole adapter, and the last loads are what their threads gave"""
    g = torch.Generator().manual_seed(670)
    d_in, d_out = 200, 300
    w = _rand(g, d_out, d_in, dtype=DT[dtype])
    layer = AdaptedProjection(w, None, 2, 32)
    x = {n: _rand(g, n, d_in, dtype=DT[dtype]).cuda() for n in (3, 700)}
    off = {n: _dev([0, n]) for n in x}
    slot = [_dev([0]), _dev([1])]
    choices = [[(_rand(g, r, d_in, dtype=DT[dtype]), _rand(g, d_out, r, dtype=DT[dtype]), 0.5) for r in (32, 7)] for _ in range(2)]
    want = {}
    for k in range(2):
        for c, ad in enumerate(choices[k]):
            layer.set_adapter(k, *ad)
            for n in x:
                want[k, c, n] = layer(x[n], off[n], slot[k])
    torch.cuda.synchronize()
    wrong, loading = [], [True, True]

    def load(k):
        try:
            for i in range(150):
                layer.set_adapter(k, *choices[k][i % 2])
        except Exception as e:                              # noqa: BLE001 (a thread's failure is the test's)
            wrong.append(repr(e))
        loading[k] = False

    def decode(n):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for i in range(3000):
                    if not any(loading):
                        break
                    k = i & 1
                    y = layer(x[n], off[n], slot[k])
                    if not any(torch.equal(y, want[k, c, n]) for c in range(2)):
                        wrong.append("%d rows, slot %d: neither adapter's result" % (n, k))
                        break
            stream.synchronize()
        except Exception as e:                              # noqa: BLE001
            wrong.append(repr(e))

    threads = [threading.Thread(target=load, args=(k,)) for k in range(2)] + [threading.Thread(target=decode, args=(n,)) for n in x]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    for k in range(2):
        for n in x:
            assert torch.equal(layer(x[n], off[n], slot[k]), want[k, 1, n])


def test_tensors_with_a_tangent_are_refused():
    import torch.autograd.forward_ad as forward
    x, w = torch.ones(6, 12, device="cuda"), torch.ones(12, device="cuda")
    layer, off = AdaptedProjection(torch.ones(8, 12)), _dev([0, 6])
    with forward.dual_level():
        dx, dw = forward.make_dual(x, torch.ones_like(x)), forward.make_dual(w, torch.ones_like(w))
        for call in (lambda: group_norm(dx, off, 3), lambda: group_norm(x, off, 3, dw), lambda: group_norm(x, off, 3, None, dw), lambda: senone_scores(dx),
                     lambda: senone_scores(x, dw), lambda: layer(dx)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        assert torch.equal(layer(dx.detach()), layer(x)) and group_norm(x, off, 3, w).shape == x.shape and senone_scores(x, w).shape == x.shape


def test_silu_keeps_32_bits_below_zero():
    """relative to the value, not to its argument: exp2 and the reciprocal are good to 2 U each, four more roundings to U each (the argument's
    own is taken back).  A gain of 0 leaves the offset as the argument, exactly; infinite offsets, and beyond the range of exp"""
    v = torch.cat([torch.linspace(-80, 40, 4096), torch.tensor([0.0, 1e-30, -1e-30, 250.0, 1e30, float("inf")])])
    n = v.numel()
    x = torch.tensor([1.0, -1.0]).repeat(n // 2)[None].cuda()
    y = group_norm(x, _dev([0, 1]), 1, torch.zeros(n, device="cuda"), v.cuda(), act="silu")[0].double().cpu()
    want = v.double() * torch.sigmoid(v.double())
    assert y[-1] == float("inf")
    assert ((y[:-1] - want[:-1]).abs() <= 8 * net_ref.U * want[:-1].abs()).all()
    far = torch.tensor([-120.0, -1e4, -3e38, -95.0])
    y = group_norm(x[:, :4].contiguous(), _dev([0, 1]), 1, torch.zeros(4, device="cuda"), far.cuda(), act="silu")[0].cpu()
    assert (y.abs() <= 95 * np.exp(-95.0)).all() and not torch.isnan(y).any()
    nan = torch.tensor([float("nan"), -float("inf")], device="cuda")
    assert torch.isnan(group_norm(x[:, :2].contiguous(), _dev([0, 1]), 1, torch.zeros(2, device="cuda"), nan, act="silu")).all()


def test_numbers_beyond_32_bits_are_refused():
    layer = AdaptedProjection(torch.zeros(8, 12), None, 2, 4)
    layer.set_adapter(0, torch.ones(2, 12), torch.ones(8, 2))
    x, off = torch.ones(6, 12, device="cuda"), _dev([0, 6])
    with pytest.raises(ValueError):
        layer.set_adapter(1 << 32, None, None)
    assert (layer(x, off, _dev([0])) == 24.0).all()
    for n in ((1 << 32) + 3, 1 << 31):
        with pytest.raises(ValueError):
            group_norm(x, off, n)
