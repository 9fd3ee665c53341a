"""The operators of an acoustic network on the device against plain implementations in 64 bits (tests/net_ref.py), with the error
bounds derived there: packed batches with empty and one-frame utterances, odd sizes, strides and alignments, rows of no utterance,
masked and non-finite outputs, streams, graphs, and the operators run together up to the search."""
import numpy as np
import pytest
import torch

import net_ref
from pocketsphinx_amd import AdaptedProjection, FwdtreeSearch, PsgpuError, group_norm, senone_scores

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _off(lens, start=0):
    return [start] + [start + int(v) for v in np.cumsum(lens)]


def _dev(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _strided(t, pad=0, shift=0):
    """t on the device in a wider buffer: row stride width + pad, `shift` elements behind an aligned address"""
    buf = torch.full((t.shape[0] * (t.shape[1] + pad) + shift + 64,), float("nan"), dtype=t.dtype, device="cuda")
    v = buf[shift:shift + t.shape[0] * (t.shape[1] + pad)].view(t.shape[0], t.shape[1] + pad)[:, :t.shape[1]]
    v.copy_(t)
    return v


def _close(got, want, err, dtype, what):
    """|got - want| within the bound; non-finite values alike"""
    got = got.detach().double().cpu()
    tol = err + net_ref.stored(want.abs() + err, dtype)
    fin = torch.isfinite(want)
    bad = torch.where(fin, ~((got - want).abs() <= tol), torch.zeros_like(fin))
    if bad.any():
        i = torch.nonzero(bad)[0].tolist()
        raise AssertionError("%s: %d of %d values off, first at %r: %r, not %r +- %r" % (what, int(bad.sum()), bad.numel(), i,
                                                                                        float(got[tuple(i)]), float(want[tuple(i)]), float(tol[tuple(i)])))


# ---- the projection ----------------------------------------------------------------------------------------------------------------

def _layer(g, dtype, d_in, d_out, ranks, max_rank, bias=True, scale=1.5):
    w = _rand(g, d_out, d_in, dtype=dtype, scale=d_in ** -0.5)
    b = _rand(g, d_out) if bias else None
    layer = AdaptedProjection(w, b, max_adapters=len(ranks), max_rank=max_rank)
    ad = {}
    for s, r in enumerate(ranks):
        if r:
            ad[s] = (_rand(g, r, d_in, dtype=dtype, scale=d_in ** -0.5), _rand(g, d_out, r, dtype=dtype), scale)
            layer.set_adapter(s, *ad[s])
    return layer, w, b, ad


PROJ = [
    # d_in, d_out, utterance lengths, slots, ranks of the slots, max_rank
    (1, 1, [1], [0], [1], 1),
    (39, 70, [1], [-1], [4], 8),
    (64, 64, [1], [0], [16], 16),
    (429, 257, [1, 2, 3, 0, 5], [0, 1, -1, 0, 1], [8, 3], 8),
    (1024, 5126, [1], [0], [16], 16),
    (1024, 1024, [1] * 70, [u % 9 - 1 for u in range(70)], [16] * 8, 16),
    (1024, 512, [10] * 33, [u % 5 - 1 for u in range(33)], [5, 0, 33, 64], 64),
    (351, 300, [0, 17, 0, 0, 130, 1, 63, 64, 65, 0], [0, 1, 2, 0, 1, 2, -1, 0, 1, 2], [16, 24, 128], 128),
    (512, 640, [300, 1, 211], [1, 0, 1], [32, 20], 32),
    (200, 129, [513, 255], [0, 7], [17], 20),
    (77, 1000, [129], None, [], 1),
    (2048, 96, [40, 24], [0, 1], [64, 1], 64),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ci", range(len(PROJ)))
def test_projection_with_adapters(ci, dtype):
    d_in, d_out, lens, slots, ranks, max_rank = PROJ[ci]
    g = torch.Generator().manual_seed(100 + ci)
    layer, w, b, ad = _layer(g, DT[dtype], d_in, d_out, ranks, max_rank, bias=ci % 3 != 1)
    off = _off(lens)
    x = _rand(g, off[-1], d_in, dtype=DT[dtype])
    want, err = net_ref.proj(x, w, b, ad, off, slots)
    got = layer(x.cuda(), _dev(off), _dev(slots) if slots is not None else None)
    assert got.dtype == DT[dtype] and got.shape == want.shape
    _close(got, want, err, DT[dtype], "y")
    if dtype != "f32":
        _close(layer(x.cuda(), _dev(off), _dev(slots) if slots is not None else None, out_dtype=torch.float32), want, err, torch.float32, "y in 32 bits")
    plain, perr = net_ref.proj(x, w, b, {}, None, None)
    _close(layer(x.cuda()), plain, perr, DT[dtype], "the shared projection alone")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens, slots", [([4], [1]), ([1, 1, 1, 1], [2, 0, 2, 1]), ([1, 2], [-1, 3]), ([2, 0, 2], [0, 1, 2]), ([5], [2])])
def test_projection_of_a_few_rows(lens, slots, dtype):
    """up to four rows and more than that; several adapters, of the largest rank, one row of no utterance behind them"""
    g = torch.Generator().manual_seed(440)
    layer, w, b, ad = _layer(g, DT[dtype], 203, 330, [128, 7, 33], 128)
    off = _off(lens)
    for extra in (0, 1):
        x = _rand(g, off[-1] + extra, 203, dtype=DT[dtype])
        want, err = net_ref.proj(x, w, b, ad, off, slots)
        out = torch.full((off[-1] + extra, 330), 5.0, dtype=DT[dtype], device="cuda")
        layer(x.cuda(), _dev(off), _dev(slots), out=out)
        _close(out[:off[-1]], want[:off[-1]], err[:off[-1]], DT[dtype], "y")
        assert (out[off[-1]:] == 5.0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d_out", [60, 100])
def test_projection_of_many_rows_to_few_outputs(d_out, dtype):
    g = torch.Generator().manual_seed(450)
    layer, w, b, ad = _layer(g, DT[dtype], 77, d_out, [20, 0, 5], 20)
    lens, slots = [9000, 1, 0, 1, 40, 8000], [0, 2, 0, 0, -1, 2]
    off = _off(lens, start=2)
    x = _rand(g, off[-1] + 3, 77, dtype=DT[dtype])
    want, err = net_ref.proj(x, w, b, ad, off, slots)
    out = torch.full((off[-1] + 3, d_out), 5.0, dtype=DT[dtype], device="cuda")
    layer(x.cuda(), _dev(off), _dev(slots), out=out)
    _close(out[2:off[-1]], want[2:off[-1]], err[2:off[-1]], DT[dtype], "y")
    assert (out[:2] == 5.0).all() and (out[off[-1]:] == 5.0).all()


def test_rows_beyond_32_bit_offsets():
    """the last rows of buffers of more than 2^31 elements: as those rows alone"""
    g = torch.Generator(device="cuda").manual_seed(22)
    n, w = 450000, 5120
    x = torch.empty((n, w), dtype=torch.float16, device="cuda")
    x[-3000:] = torch.randn(3000, w, generator=g, device="cuda").half()
    x[:-3000] = 0.5
    off = _dev([0, n - 3000, n - 1000, n])
    assert n * w > 1 << 31
    few = senone_scores(x[-3000:], want_best=True)
    s, b = senone_scores(x, want_best=True)
    assert torch.equal(s[-3000:], few[0]) and torch.equal(b[-3000:], few[1])
    del s, b
    few = group_norm(x[-3000:], _dev([0, 2000, 3000]), 32, act="silu").double()
    y = group_norm(x, off, 32, act="silu")
    # a step of float16, and twice what either may be off before its rounding: 1.2 * 5 u |z| + 8 u |z|, |z| below 8
    assert ((y[-3000:].double() - few).abs() <= 2.0 ** -10 * few.abs() + 2 * 14 * net_ref.U * 8).all()
    del y
    layer = AdaptedProjection(torch.randn(64, w, generator=g, device="cuda").half() * w ** -0.5, None, 1, 8)
    layer.set_adapter(0, torch.randn(8, w, generator=g, device="cuda").half() * w ** -0.5, torch.randn(64, 8, generator=g, device="cuda").half())
    y = layer(x, off, _dev([-1, 0, -1]), out_dtype=torch.float32)
    few = layer(x[-3000:], _dev([0, 2000, 3000]), _dev([0, -1]), out_dtype=torch.float32)
    assert ((y[-3000:] - few).abs() <= 2 * 2 * net_ref.U * (w + 26) * 100).all()       # two orders of one sum, of magnitudes below 100


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad, shift", [(1, 0), (0, 1), (3, 5), (8, 8), (64, 0)])
@pytest.mark.parametrize("rows", [3, 150])
def test_projection_strides_and_alignment(rows, pad, shift, dtype):
    g = torch.Generator().manual_seed(7)
    layer, w, b, ad = _layer(g, DT[dtype], 130, 90, [9, 12], 12)
    off, slots = [0, rows // 3, rows], [1, 0]
    x = _rand(g, rows, 130, dtype=DT[dtype])
    want, err = net_ref.proj(x, w, b, ad, off, slots)
    out = _strided(torch.full((rows, 90), 7.0, dtype=DT[dtype]), pad, shift)
    wide = out.as_strided((rows, 90 + pad), (90 + pad, 1)) if pad else None
    keep = wide[:, 90:].clone() if pad else None
    r = layer(_strided(x, pad, shift), _dev(off), _dev(slots), out=out)
    assert r is out
    _close(out, want, err, DT[dtype], "y")
    if pad:
        assert torch.equal(torch.nan_to_num(wide[:, 90:]), torch.nan_to_num(keep)), "elements behind a row were written"


@pytest.mark.parametrize("rows", [12, 400])
def test_projection_leaves_rows_of_no_utterance(rows):
    g = torch.Generator().manual_seed(8)
    layer, w, b, ad = _layer(g, torch.bfloat16, 96, 200, [8], 8)
    x = _rand(g, rows, 96, dtype=torch.bfloat16)
    off, slots = [3, 3, 7, rows - 4], [0, -1, 0]
    out = torch.full((rows, 200), 5.0, dtype=torch.bfloat16, device="cuda")
    layer(x.cuda(), _dev(off), _dev(slots), out=out)
    want, err = net_ref.proj(x, w, b, ad, off, slots)
    _close(out[3:rows - 4], want[3:rows - 4], err[3:rows - 4], torch.bfloat16, "y")
    assert (out[:3] == 5.0).all() and (out[rows - 4:] == 5.0).all()
    # no utterance at all, offsets that reach beyond the rows, no rows
    out.fill_(5.0)
    layer(x.cuda(), _dev([0]), _dev([]), out=out)
    assert (out == 5.0).all()
    layer(x.cuda(), _dev([-9, rows + 50]), _dev([0]), out=out)
    want, err = net_ref.proj(x, w, b, ad, [-9, rows + 50], [0])
    _close(out, want, err, torch.bfloat16, "y")
    assert layer(x.cuda()[:0], _dev([0, 0]), _dev([0])).shape == (0, 200)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_projection_adapter_slots(dtype):
    """slots that name nothing, an adapter replaced, emptied, of another rank; the same slot for several utterances"""
    g = torch.Generator().manual_seed(9)
    layer, w, b, ad = _layer(g, DT[dtype], 100, 150, [5, 0, 30], 40)
    off = _off([4, 30, 1, 7, 20, 2])
    x = _rand(g, off[-1], 100, dtype=DT[dtype])
    for slots in ([0, 2, 0, 2, 2, 0], [1, 3, -1, -7, 1 << 30, -(1 << 31)], [2, 1, 0, 3, 2, 1]):
        want, err = net_ref.proj(x, w, b, ad, off, slots)
        _close(layer(x.cuda(), _dev(off), _dev(slots)), want, err, DT[dtype], "slots %r" % (slots,))
    ad[0] = (_rand(g, 11, 100, dtype=DT[dtype], scale=0.1), _rand(g, 150, 11, dtype=DT[dtype]), -0.25)
    layer.set_adapter(0, *ad[0])
    layer.set_adapter(2, None, None)
    del ad[2]
    slots = [0, 2, 0, 2, 1, 0]
    want, err = net_ref.proj(x, w, b, ad, off, slots)
    _close(layer(x.cuda(), _dev(off), _dev(slots)), want, err, DT[dtype], "after the change")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_projection_keeps_other_rows_from_non_finite_ones(dtype):
    """an infinity or a NaN in one row stays in that row; the rows behind a non-finite one in its tile are as ever"""
    g = torch.Generator().manual_seed(10)
    layer, w, b, ad = _layer(g, DT[dtype], 75, 60, [4, 6], 8)
    off, slots = _off([1, 40, 3]), [0, 1, 0]
    x = _rand(g, off[-1], 75, dtype=DT[dtype])
    want, err = net_ref.proj(x, w, b, ad, off, slots)
    x[7, 74] = float("inf"); x[0, 0] = float("nan"); x[42, 30] = float("-inf")
    got = layer(x.cuda(), _dev(off), _dev(slots)).double().cpu()
    mask = torch.ones(off[-1], dtype=torch.bool)
    mask[[0, 7, 42]] = False
    _close(got[mask], want[mask], err[mask], DT[dtype], "finite rows")
    assert torch.isnan(got[0]).all() and not torch.isfinite(got[7]).any() and not torch.isfinite(got[42]).any()
    plain = layer(x.cuda()).double().cpu()
    assert torch.equal(plain[7], torch.sign(w[:, 74].double()) * float("inf")), "an infinity times a weight"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_projection_large_hidden_values(dtype):
    """h beyond a half's range: the adapter's sum is still a number"""
    g = torch.Generator().manual_seed(11)
    layer = AdaptedProjection(torch.zeros(33, 64, dtype=DT[dtype]), None, max_adapters=1, max_rank=4)
    a, b = torch.full((4, 64), 40.0, dtype=DT[dtype]), _rand(g, 33, 4, dtype=DT[dtype], scale=2.0 ** -14)
    layer.set_adapter(0, a, b, 1.0)
    x = torch.full((20, 64), 60.0, dtype=DT[dtype])
    want, err = net_ref.proj(x, torch.zeros(33, 64), None, {0: (a, b, 1.0)}, [0, 20], [0])
    _close(layer(x.cuda(), _dev([0, 20]), _dev([0])), want, err, DT[dtype], "y")


LARGE = [
    # d_in, d_out, rows (about), elements behind a row: tiles of 128 and of 256 frames, x aligned to 16 bytes or not, a last stage that d_in
    # does not fill (136 = 2 * 64 + 8) or does (128), a d_in below one stage
    (136, 5126, 1000, 0),
    (101, 5126, 1000, 3),
    (128, 2100, 2500, 8),
    (136, 5126, 6500, 0),
    (128, 5126, 6500, 1),
    (136, 5126, 1000, 2),
    (150, 5126, 6500, 6),
    (24, 8192, 4300, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ci", range(len(LARGE)))
def test_projection_in_large_tiles(ci, dtype):
    """many frames: tiles with one adapter, with several, with frames of one-frame utterances, frames of no utterance"""
    d_in, d_out, rows, pad = LARGE[ci]
    g = torch.Generator().manual_seed(400 + ci)
    layer, w, b, ad = _layer(g, DT[dtype], d_in, d_out, [16, 0, 40, 3], 40)
    lens = [rows // 3, 1, 1, 0, 1, 17, rows // 5, 2, 2, 0, 0, 1]
    off = _off(lens + [rows // 4], start=5)
    n = off[-1] + 9
    slots = [0, 2, 0, 1, 3, -1, 2, 3, 0, 2, 2, -1, 3]
    x = _rand(g, n, d_in, dtype=DT[dtype])
    want, err = net_ref.proj(x, w, b, ad, off, slots)
    out = torch.full((n, d_out), 5.0, dtype=DT[dtype], device="cuda")
    layer(_strided(x, pad), _dev(off), _dev(slots), out=out)
    _close(out[5:off[-1]], want[5:off[-1]], err[5:off[-1]], DT[dtype], "y")
    assert (out[:5] == 5.0).all() and (out[off[-1]:] == 5.0).all()
    if dtype != "f32":
        _close(layer(_strided(x, pad), _dev(off), _dev(slots), out_dtype=torch.float32)[5:off[-1]], want[5:off[-1]], err[5:off[-1]], torch.float32, "y in 32 bits")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 2, 3])
@pytest.mark.parametrize("rows, d_in, d_out", [(20000, 1000, 2100), (4300, 1024, 8192), (2500, 2048, 1024)])
def test_projection_over_many_stages(rows, d_in, d_out, pad, dtype):
    """a long reduced axis in large tiles: every stage is whole before it is multiplied (64-bit products on the device)"""
    g = torch.Generator().manual_seed(430)
    layer, w, b, ad = _layer(g, DT[dtype], d_in, d_out, [24, 7], 24)
    off, slots = [0, rows // 2 + 3, rows], [0, 1]
    x = _rand(g, rows, d_in, dtype=DT[dtype])
    xd, wd = x.cuda().double(), w.cuda().double()
    want = xd @ wd.t() + b.cuda().double()
    mag = xd.abs() @ wd.abs().t() + b.cuda().double().abs()
    err = torch.zeros_like(want)
    for u, s in enumerate(slots):               # as net_ref.proj
        a, bb, sc = (v.cuda().double() if torch.is_tensor(v) else v for v in ad[s])
        r = slice(off[u], off[u + 1])
        h = sc * (xd[r] @ a.t())
        want[r] += h @ bb.t()
        mag[r] += h.abs() @ bb.abs().t()
        err[r] = (sc * (xd[r].abs() @ a.abs().t()) * (2 * net_ref.U * (d_in + 1)) + h.abs() * (2.0 ** -16 + 2.0 ** -17)) @ bb.abs().t()
        err[r] += 2 * net_ref.U * (d_in + 1 + 3 * a.shape[0]) * mag[r]
    want, err = want.cpu(), err.cpu()
    xs = _strided(x, pad)
    for _ in range(3):
        _close(layer(xs, _dev(off), _dev(slots)), want, err, DT[dtype], "y")


def test_projection_keeps_other_rows_from_non_finite_ones_in_large_tiles():
    g = torch.Generator().manual_seed(410)
    layer, w, b, ad = _layer(g, torch.bfloat16, 136, 5126, [4, 6], 8)
    off, slots = _off([1, 400, 900]), [0, 1, 0]
    x = _rand(g, off[-1], 136, dtype=torch.bfloat16)
    want, err = net_ref.proj(x, w, b, ad, off, slots)
    x[7, 135] = float("inf"); x[0, 0] = float("nan"); x[1300, 30] = float("-inf")
    got = layer(x.cuda(), _dev(off), _dev(slots)).double().cpu()
    mask = torch.ones(off[-1], dtype=torch.bool)
    mask[[0, 7, 1300]] = False
    _close(got[mask], want[mask], err[mask], torch.bfloat16, "finite rows")
    assert torch.isnan(got[0]).all() and not torch.isfinite(got[7]).any() and not torch.isfinite(got[1300]).any()


@pytest.mark.parametrize("lens", [[1] * 300, [0] * 200 + [1] * 3 + [0] * 500 + [2] * 70, [1] * 5000, [0, 0, 1]])
def test_projection_finds_the_utterance_of_every_row(lens):
    """many utterances, runs of empty ones: each row its own adapter's factor"""
    layer = AdaptedProjection(torch.zeros(16, 8), None, max_adapters=97, max_rank=1)
    for s in range(97):
        layer.set_adapter(s, torch.ones(1, 8), torch.ones(16, 1), float(s + 1))
    off = _off(lens)
    slots = [(31 * u) % 97 for u in range(len(lens))]
    y = layer(torch.ones(off[-1], 8, device="cuda"), _dev(off), _dev(slots)).cpu()
    want = torch.tensor([8.0 * (slots[u] + 1) for u, n in enumerate(lens) for _ in range(n)])
    assert torch.equal(y, want[:, None].expand(-1, 16))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_projection_takes_weights_from_the_device(dtype):
    g = torch.Generator().manual_seed(420)
    w, b = _rand(g, 70, 40, dtype=DT[dtype]), _rand(g, 70)
    a, bb = _rand(g, 5, 40, dtype=DT[dtype]), _rand(g, 70, 5, dtype=DT[dtype])
    one, two = AdaptedProjection(w, b, 1, 8), AdaptedProjection(w.cuda(), b.cuda(), 1, 8)
    one.set_adapter(0, a, bb, 0.5)
    two.set_adapter(0, a.cuda(), bb.t().contiguous().cuda().t(), 0.5)
    x = _rand(g, 33, 40, dtype=DT[dtype]).cuda()
    assert torch.equal(one(x, _dev([0, 33]), _dev([0])), two(x, _dev([0, 33]), _dev([0])))


def test_projection_refusals():
    w = torch.zeros(8, 16, dtype=torch.bfloat16)
    layer = AdaptedProjection(w, None, max_adapters=2, max_rank=4)
    x = torch.zeros(5, 16, dtype=torch.bfloat16, device="cuda")
    for bad in (x.float(), x[:, :15], x.cpu(), x[0], x.t().contiguous().t(), x[:1].expand(5, 16)):
        with pytest.raises(ValueError):
            layer(bad)
    off = _dev([0, 5])
    for kw in (dict(adapter=_dev([0])), dict(utt_off=off.long(), adapter=_dev([0])), dict(utt_off=off, adapter=_dev([0, 1])), dict(utt_off=off.cpu()),
               dict(out=torch.zeros(5, 8, device="cuda", dtype=torch.float16)), dict(out=torch.zeros(4, 8, device="cuda")), dict(out_dtype=torch.float16)):
        with pytest.raises(ValueError):
            layer(x, **kw)
    with pytest.raises(PsgpuError):
        layer(x, out=x[:, :8])
    for s, a, b in ((2, torch.zeros(2, 16), torch.zeros(8, 2)), (-1, torch.zeros(2, 16), torch.zeros(8, 2)), (0, torch.zeros(5, 16), torch.zeros(8, 5))):
        with pytest.raises(PsgpuError):
            layer.set_adapter(s, a.bfloat16(), b.bfloat16())
    with pytest.raises(PsgpuError):
        layer.set_adapter(0, torch.zeros(2, 16).bfloat16(), torch.zeros(8, 2).bfloat16(), float("nan"))
    for a, b in ((torch.zeros(2, 16), torch.zeros(8, 2)), (torch.zeros(2, 15).bfloat16(), torch.zeros(8, 2).bfloat16()),
                 (torch.zeros(2, 16).bfloat16(), torch.zeros(8, 3).bfloat16()), (torch.zeros(2, 16).bfloat16(), None)):
        with pytest.raises(ValueError):
            layer.set_adapter(0, a, b)
    with pytest.raises(PsgpuError):
        AdaptedProjection(w, None, max_adapters=1, max_rank=129)
    with pytest.raises(ValueError):
        AdaptedProjection(w, torch.zeros(7))
    with pytest.raises(ValueError):
        AdaptedProjection(w.double())


# ---- group norm --------------------------------------------------------------------------------------------------------------------

GN = [
    # lengths, channels, groups, activation, eps
    ([1], 1, 1, "none", 1e-5),
    ([1], 1024, 32, "silu", 1e-5),
    ([1, 0, 2, 3], 39, 3, "relu", 1e-5),
    ([10] * 40, 256, 8, "gelu", 1e-5),
    ([0, 0, 700, 1, 33, 0], 429, 11, "silu", 1e-3),
    ([900, 257], 130, 1, "none", 1e-5),
    ([64, 65, 63], 96, 96, "gelu", 1e-5),
    ([5, 3000], 64, 2, "relu", 1e-5),
    ([300], 2048, 16, "silu", 1e-5),
    ([1200, 1], 1030, 5, "gelu", 0.0),
    ([7, 2], 5000, 1, "none", 1e-5),
    ([40, 30, 2], 6000, 1, "silu", 1e-5),
    ([40, 0, 30, 2], 12002, 2, "gelu", 1e-5),
    ([3300, 1, 700, 0, 45, 2, 90, 1300, 30, 31, 32, 33, 34, 64, 65, 129], 1024, 32, "gelu", 1e-5),
    ([129, 130, 400, 1] * 2, 2048, 64, "relu", 1e-5),
    ([2, 0, 5, 1, 9] * 60, 301, 43, "silu", 1e-5),
    ([1] * 512, 17000, 1, "none", 1e-5),
    ([3000, 0, 1, 2, 70, 13000], 512, 128, "silu", 1e-5),
    ([3000, 0, 5000, 1, 14000, 700], 1024, 128, "gelu", 1e-5),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ci", range(len(GN)))
def test_group_norm(ci, dtype):
    lens, chan, groups, name, eps = GN[ci]
    if eps == 0.0:
        lens = [n for n in lens if n > 1]
    g = torch.Generator().manual_seed(200 + ci)
    off = _off(lens)
    x = (_rand(g, off[-1], chan) * torch.exp(_rand(g, chan, scale=0.5)) + _rand(g, chan, scale=2.0)).to(DT[dtype])
    w, b = (1 + _rand(g, chan, scale=0.3), _rand(g, chan, scale=0.5)) if ci % 3 else (None, None)
    want, err = net_ref.gnorm(x, off, groups, w, b, float(np.float32(eps)), name)
    dw, db = (None, None) if w is None else (w.cuda(), b.cuda())
    got = group_norm(x.cuda(), _dev(off), groups, dw, db, eps=eps, act=name)
    assert got.dtype == DT[dtype] and got.shape == x.shape
    _close(got, want, err, DT[dtype], "y")
    xd = x.cuda()
    assert group_norm(xd, _dev(off), groups, dw, db, eps=eps, act=name, out=xd) is xd
    assert torch.equal(xd.view(torch.int32 if dtype == "f32" else torch.int16), got.view(torch.int32 if dtype == "f32" else torch.int16)), "in place"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad, shift", [(1, 0), (0, 1), (3, 5), (8, 0)])
@pytest.mark.parametrize("lens", [[2, 3], [150, 0, 31]])
def test_group_norm_strides_and_alignment(lens, pad, shift, dtype):
    g = torch.Generator().manual_seed(12)
    off = _off(lens)
    x = _rand(g, off[-1], 104, dtype=DT[dtype])
    w, b = 1 + _rand(g, 104, scale=0.3), _rand(g, 104)
    want, err = net_ref.gnorm(x, off, 8, w, b, float(np.float32(1e-5)), "silu")
    out = _strided(torch.full((off[-1], 104), 7.0, dtype=DT[dtype]), pad, shift)
    wide = out.as_strided((off[-1], 104 + pad), (104 + pad, 1)) if pad else None
    keep = wide[:, 104:].clone() if pad else None
    group_norm(_strided(x, pad, shift), _dev(off), 8, w.cuda(), b.cuda(), act="silu", out=out)
    _close(out, want, err, DT[dtype], "y")
    if pad:
        assert torch.equal(torch.nan_to_num(wide[:, 104:]), torch.nan_to_num(keep)), "elements behind a row were written"


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_tensors_that_ask_for_a_gradient_are_refused(dtype):
    x = torch.zeros(6, 12, dtype=DT[dtype], device="cuda", requires_grad=True)
    w = torch.zeros(12, device="cuda", requires_grad=True)
    layer = AdaptedProjection(torch.zeros(8, 12, dtype=DT[dtype], requires_grad=True))
    off = _dev([0, 6])
    for call in (lambda: group_norm(x, off, 3), lambda: group_norm(x.detach(), off, 3, w), lambda: senone_scores(x), lambda: layer(x)):
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():
        assert group_norm(x, off, 3, w).shape == x.shape and senone_scores(x).shape == x.shape and layer(x).shape == (6, 8)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_group_norm_rows_far_apart(dtype):
    g = torch.Generator().manual_seed(21)
    off = [0, 3, 20]
    x = _rand(g, 20, 64, dtype=DT[dtype])
    want, err = net_ref.gnorm(x, off, 4, None, None, float(np.float32(1e-5)), "gelu")
    out = _strided(torch.full((20, 64), 7.0, dtype=DT[dtype]), 70001)
    group_norm(_strided(x, 65536), _dev(off), 4, act="gelu", out=out)
    _close(out, want, err, DT[dtype], "y")


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_group_norm_activations_over_their_range(act):
    """values from -40 to 40 through the activation: a group of two far values keeps the others' places (bias alone moves them)"""
    x = torch.tensor([[1.0, -1.0]]).repeat(4001, 1)
    b = torch.linspace(-40, 40, 4001)
    y = torch.cat([group_norm(x[:1].cuda(), _dev([0, 1]), 1, torch.zeros(2, device="cuda"), torch.tensor([float(v), float(v)], device="cuda"), act=act) for v in b[::40]])
    want = net_ref.act(act, b[::40].double())
    _close(y[:, 0], want, 9 * net_ref.U * b[::40].double().abs(), torch.float32, act)


def test_group_norm_leaves_rows_of_no_utterance():
    g = torch.Generator().manual_seed(13)
    for rows, off in ((30, [4, 4, 9, 20]), (600, [1, 300, 598]), (30, [30, 30]), (30, [-5, 12, 90])):
        x = _rand(g, rows, 64)
        out = torch.full((rows, 64), 5.0, device="cuda")
        group_norm(x.cuda(), _dev(off), 4, act="none", out=out)
        want, err = net_ref.gnorm(x, off, 4, None, None, float(np.float32(1e-5)), "none")
        inside = ~torch.isnan(want[:, 0])
        _close(out[inside.cuda()], want[inside], err[inside], torch.float32, "y")
        assert (out[~inside.cuda()] == 5.0).all()
    x = torch.ones(4, 8, device="cuda")
    assert (group_norm(x, _dev([0]), 2, out=torch.full((4, 8), 5.0, device="cuda")) == 5.0).all()
    assert group_norm(x[:0], _dev([0, 0]), 2).shape == (0, 8)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [4, 800])
def test_group_norm_far_means_constants_and_non_finite_values(rows, dtype):
    """a mean far above the spread; a group without spread (act(bias)); a NaN and an infinity make their utterance's group NaN and no other"""
    g = torch.Generator().manual_seed(14)
    x = _rand(g, 2 * rows, 24)
    x[:, :8] = x[:, :8] * 4 + 1e4                  # group 0
    x[:, 8:16] = 3.25                              # group 1
    x = x.to(DT[dtype])
    b = _rand(g, 24)
    off = [0, rows, 2 * rows]
    want, err = net_ref.gnorm(x, off, 3, None, b, float(np.float32(1e-5)), "none")
    got = group_norm(x.cuda(), _dev(off), 3, None, b.cuda())
    _close(got, want, err, DT[dtype], "y")
    assert torch.equal(got[:, 8:16].cpu(), b[8:16].to(DT[dtype]).expand(2 * rows, 8))
    x[1, 17] = float("nan"); x[rows + 1, 2] = float("inf")
    got = group_norm(x.cuda(), _dev(off), 3, None, b.cuda()).cpu()
    nan = torch.zeros(2 * rows, 24, dtype=torch.bool)
    nan[:rows, 16:] = True; nan[rows:, :8] = True
    assert torch.equal(torch.isnan(got), nan)
    _close(got.double()[~nan], want[~nan], err[~nan], DT[dtype], "the other groups")


def test_group_norm_large_values():
    """values whose squares pass float32's range"""
    x = torch.tensor([[3e30, -3e30, 1e30, 0.0]], device="cuda")
    want, err = net_ref.gnorm(x, [0, 1], 1, None, None, float(np.float32(1e-5)), "none")
    _close(group_norm(x, _dev([0, 1]), 1), want, err, torch.float32, "y")


def test_group_norm_refusals():
    x, off = torch.zeros(6, 12, device="cuda"), _dev([0, 6])
    for kw in (dict(n_groups=5), dict(n_groups=0), dict(n_groups=-3), dict(n_groups=24), dict(n_groups=3, eps=-1.0), dict(n_groups=3, eps=float("nan"))):
        with pytest.raises(PsgpuError):
            group_norm(x, off, **kw)
    w = torch.zeros(12, device="cuda")
    for a, kw in ((x.cpu(), {}), (x.double(), {}), (x, dict(weight=w[:11])), (x, dict(bias=w.half())), (x, dict(weight=w.cpu())), (x, dict(act="tanh")),
                  (x, dict(out=torch.zeros(6, 12, device="cuda", dtype=torch.float16))), (x, dict(out=torch.zeros(5, 12, device="cuda")))):
        with pytest.raises(ValueError):
            group_norm(a, off, 3, **kw)
    big = torch.zeros(13, 12, device="cuda")
    with pytest.raises(PsgpuError):
        group_norm(big[:6], off, 3, out=big[1:7])


# ---- senone scores -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows, n_sen", [(1, 1), (1, 5126), (3, 7), (40, 5126), (65, 127), (2, 20000), (9, 2049), (300, 100)])
def test_senone_scores(rows, n_sen, dtype):
    g = torch.Generator().manual_seed(300 + rows + n_sen)
    z = _rand(g, rows, n_sen, dtype=DT[dtype], scale=4.0)
    prior = torch.log_softmax(_rand(g, n_sen).double(), 0).float()
    for p, scale, base in ((prior, 0.8, 1.0001), (None, 1.0, 1.0001), (prior, 300.0, 1.0003)):
        ws, wb, be = net_ref.senones(z, p, scale, base)
        s, b = senone_scores(z.cuda(), None if p is None else p.cuda(), scale=scale, logbase=base, want_best=True)
        assert s.dtype == torch.int16 and np.array_equal(s.cpu().numpy(), ws)
        assert (np.abs(b.double().cpu().numpy() - wb) <= be).all()
        assert torch.equal(senone_scores(z.cuda(), None if p is None else p.cuda(), scale=scale, logbase=base), s)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows, n_sen", [(600, 100), (1500, 2050), (530, 5126), (520, 3500), (515, 8190), (3, 45000), (600, 5)])
def test_senone_scores_of_many_rows_and_long_ones(rows, n_sen, dtype):
    """with masked senones, NaN, infinities and rows of nothing in between"""
    g = torch.Generator().manual_seed(500 + n_sen)
    z = _rand(g, rows, n_sen, dtype=DT[dtype], scale=4.0)
    inf, k = float("inf"), rows // 3
    z[0, 1:] = -inf
    z[1] = -inf
    z[2] = torch.finfo(DT[dtype]).min
    if k > 2:
        z[k] = float("nan"); z[k + 1, ::3] = -inf; z[k + 2, n_sen - 1] = float("nan"); z[k + 3, n_sen // 2] = inf; z[k + 4, 0] = torch.finfo(DT[dtype]).max
    prior = torch.log_softmax(_rand(g, n_sen).double(), 0).float()
    ws, wb, be = net_ref.senones(z, prior, 0.8, 1.0001)
    s, b = senone_scores(z.cuda(), prior.cuda(), scale=0.8, want_best=True)
    assert np.array_equal(s.cpu().numpy(), ws)
    b = b.double().cpu().numpy()
    fin = np.isfinite(wb)
    assert (np.abs(b[fin] - wb[fin]) <= be[fin] + np.abs(wb[fin]) * 2.0 ** -22).all()
    assert b[1] == -inf and (k <= 2 or (np.isnan(b[k]) and np.isnan(b[k + 2])))


@pytest.mark.parametrize("pad, shift", [(1, 0), (0, 1), (3, 5), (8, 0)])
def test_senone_scores_strides(pad, shift):
    g = torch.Generator().manual_seed(15)
    z = _rand(g, 20, 333, dtype=torch.float16, scale=4.0)
    ws, _, _ = net_ref.senones(z, None, 1.0, 1.0001)
    wide = torch.full((20 * (333 + pad) + shift,), -5, dtype=torch.int16, device="cuda")
    out = wide[shift:].view(20, 333 + pad)[:, :333]
    senone_scores(_strided(z, pad, shift), out=out)
    assert np.array_equal(out.cpu().numpy(), ws)
    out.fill_(-5)
    assert (wide == -5).all(), "elements behind a row were written"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_sen", [9, 3001])
def test_senone_scores_masked_and_non_finite(n_sen, dtype):
    """-inf masks a senone; a row of nothing else has no best; NaN counts as -inf and shows in best; +inf is the best; the type's
    lowest value is a value"""
    g = torch.Generator().manual_seed(16)
    z = _rand(g, 8, n_sen, dtype=DT[dtype], scale=3.0)
    inf = float("inf")
    z[0, ::2] = -inf
    z[1] = -inf
    z[2, 3] = float("nan")
    z[3, 5] = inf
    z[4, 1:] = torch.finfo(DT[dtype]).min
    z[5] = torch.finfo(DT[dtype]).min
    z[6] = float("nan")
    z[7, 4:] = -inf
    prior = _rand(g, n_sen)
    ws, wb, be = net_ref.senones(z, prior, 1.0, 1.0001)
    s, b = senone_scores(z.cuda(), prior.cuda(), want_best=True)
    s, b = s.cpu().numpy(), b.double().cpu().numpy()
    assert np.array_equal(s, ws)
    assert (s[1] == 32767).all() and (s[6] == 32767).all() and (s[0, ::2] == 32767).all() and s[2, 3] == 32767 and s[3, 5] == 0
    assert b[1] == -inf and np.isnan(b[2]) and np.isnan(b[6])
    for r in (0, 4, 5, 7):
        assert abs(b[r] - wb[r]) <= be[r] + abs(wb[r]) * 2.0 ** -22


def test_senone_scores_refusals():
    z = torch.zeros(4, 10, device="cuda")
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(logbase=1.0), dict(logbase=0.5), dict(logbase=float("nan"))):
        with pytest.raises(PsgpuError):
            senone_scores(z, **kw)
    for a, kw in ((z.cpu(), {}), (z.double(), {}), (z, dict(log_prior=torch.zeros(9, device="cuda"))), (z, dict(log_prior=torch.zeros(10))),
                  (z, dict(out=torch.zeros(4, 10, device="cuda"))), (z, dict(out=torch.zeros(3, 10, device="cuda", dtype=torch.int16)))):
        with pytest.raises(ValueError):
            senone_scores(a, **kw)
    with pytest.raises(PsgpuError):
        senone_scores(z, out=z.view(torch.int16)[:, :10])
    assert senone_scores(z[:0]).shape == (0, 10)


# ---- together ----------------------------------------------------------------------------------------------------------------------

def _network(g, dtype, d_in, hidden, n_sen, n_adapters):
    first, w1, b1, ad1 = _layer(g, dtype, d_in, hidden, [8] * n_adapters, 8)
    last, w2, b2, ad2 = _layer(g, dtype, hidden, n_sen, [8] * n_adapters, 8)
    gw, gb = 1 + _rand(g, hidden, scale=0.2), _rand(g, hidden, scale=0.2)
    prior = torch.log_softmax(_rand(g, n_sen).double(), 0).float()
    dgw, dgb, dp = gw.cuda(), gb.cuda(), prior.cuda()

    def run(x, off, slots):
        h = group_norm(first(x, off, slots), off, 16, dgw, dgb, act="silu")
        z = last(h, off, slots, out_dtype=torch.float32)
        return h, z, senone_scores(z, dp, scale=0.5, want_best=True)
    return run, (w1, b1, ad1, gw, gb, w2, b2, ad2, prior)


@pytest.mark.parametrize("lens", [[1, 1, 1, 1], [37, 0, 120, 1, 64]])
def test_a_network_from_features_to_senone_scores(lens):
    """the operators in a row, each step held against the 64-bit form of its own input"""
    g = torch.Generator().manual_seed(17)
    run, (w1, b1, ad1, gw, gb, w2, b2, ad2, prior) = _network(g, torch.bfloat16, 117, 256, 500, 3)
    off = _off(lens)
    slots = [u % 4 - 1 for u in range(len(lens))]
    x = _rand(g, off[-1], 117, dtype=torch.bfloat16)
    h, z, (s, best) = run(x.cuda(), _dev(off), _dev(slots))
    y, err = net_ref.proj(x, w1, b1, ad1, off, slots)
    first = AdaptedProjection(w1, b1, max_adapters=3, max_rank=8)
    for k, v in ad1.items():
        first.set_adapter(k, *v)
    y1 = first(x.cuda(), _dev(off), _dev(slots))
    _close(y1, y, err, torch.bfloat16, "first layer")
    wh, herr = net_ref.gnorm(y1.cpu(), off, 16, gw, gb, float(np.float32(1e-5)), "silu")
    _close(h, wh, herr, torch.bfloat16, "norm")
    wz, zerr = net_ref.proj(h.cpu(), w2, b2, ad2, off, slots)
    _close(z, wz, zerr, torch.float32, "outputs")
    ws, wb, be = net_ref.senones(z.cpu(), prior, 0.5, 1.0001)
    assert np.array_equal(s.cpu().numpy(), ws)
    assert (np.abs(best.double().cpu().numpy() - wb) <= be).all()


def test_a_network_on_another_stream_and_in_a_graph():
    """the whole run on a side stream, captured and replayed with other inputs, eager work between the replays; two graphs at once"""
    g = torch.Generator().manual_seed(18)
    run, _ = _network(g, torch.float16, 117, 256, 500, 3)
    lens, slots = [5, 0, 130, 1, 31], [0, 1, -1, 2, 1]
    off, sl = _dev(_off(lens)), _dev(slots)
    xs = [_rand(g, sum(lens), 117, dtype=torch.float16).cuda() for _ in range(4)]
    want = [[t.clone() for t in (lambda r: (r[0], r[1], r[2][0], r[2][1]))(run(x, off, sl))] for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h, z, (s, b) = run(xs[0], off, sl)
    side.synchronize()
    for got, w in zip((h, z, s, b), want[0]):
        assert torch.equal(got, w)
    graphs = []
    for _ in range(2):
        buf = xs[0].clone()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            h, z, (s, b) = run(buf, off, sl)
        graphs.append((gr, buf, (h, z, s, b)))
    s2 = torch.cuda.Stream()
    for i in range(4):
        for (gr, buf, _), k in zip(graphs, (i, 3 - i)):
            buf.copy_(xs[k])
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(s2):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for (gr, buf, outs), k in zip(graphs, (i, 3 - i)):
            for got, w in zip(outs, want[k]):
                assert torch.equal(got, w)
        run(xs[i], off, sl)
        torch.cuda.synchronize()


def test_results_do_not_change_from_call_to_call():
    """no atomics whose order changes results: ten calls, one answer, and a frame's answer does not hang on its neighbours"""
    g = torch.Generator().manual_seed(19)
    run, _ = _network(g, torch.bfloat16, 200, 320, 700, 3)
    lens = [700, 3, 1500]
    off, sl = _dev(_off(lens)), _dev([0, 1, 2])
    x = _rand(g, sum(lens), 200, dtype=torch.bfloat16).cuda()
    first = run(x, off, sl)
    for _ in range(9):
        again = run(x, off, sl)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1]) and torch.equal(first[2][0], again[2][0]) and torch.equal(first[2][1], again[2][1])


def test_the_search_decodes_from_a_networks_outputs():
    """an output layer whose outputs are a recording's senone log-likelihoods plus priors: the layer and the scores give the
    recording's score rows back (each over its frame's best), and the tree search on the device leaves the reference's tables"""
    from test_oracle_golden import _load
    from test_search_gpu import _check, _inputs
    g = _load("fwdtree_trace_goforward_after_numbers.npz")
    search = FwdtreeSearch(_load("fwdtree_static_en_us_turtle.npz"), g["par"])
    rows, pen = _inputs(g, search.n_sen)
    rng = np.random.default_rng(20)
    raw = rng.integers(0, 3000, rows.shape)        # what the search does not ask for: anything above the frame's best
    off, act = g["step_act_off"], g["step_act"]
    for i in range(rows.shape[0]):
        raw[i, act[off[i]:off[i + 1]]] = rows[i, act[off[i]:off[i + 1]]]
    raw += rng.integers(-3000, 3000, (rows.shape[0], 1))
    gen = torch.Generator().manual_seed(20)
    prior = torch.log_softmax(_rand(gen, search.n_sen).double(), 0).float()
    loglike = torch.from_numpy(-(raw.astype(np.float64) * (np.log(1.0001) * 1024))).float()
    layer = AdaptedProjection(torch.eye(search.n_sen), prior)
    scores = senone_scores(layer(loglike.cuda()), prior.cuda())
    want = (raw - raw.min(axis=1, keepdims=True)).astype(np.int16)
    assert np.array_equal(scores.cpu().numpy(), want)
    _check(search.search(scores, pen, [rows.shape[0]], raw_scores=True, pl_window=0, mpx_in=g["mpx_init"][None])[0], g, "from the network's scores")
    search.close()
