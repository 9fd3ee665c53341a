"""The operators of an acoustic network beside the decoder -- a shared projection with low-rank adapters of many utterances, group norm
with an activation over packed utterances, senone scores of a network's outputs -- as cases to be timed and compared: their inputs,
their plain forms in elementary torch operations, their definitions in 64 bits, and the calls a user makes of the framework.

Rows are frames of utterances back to back; utterance u is rows off[u] .. off[u + 1] - 1, as everywhere in this framework."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
LOGBASE = 1.0001                        # the decoder's -logbase
SENSCR_SHIFT = 10


# ---- cases -------------------------------------------------------------------------------------------------------------------------

def listed():
    """Frames come 100 a second: 2998 are 30 s of audio, 10 are what a live stream brings each 100 ms."""
    return [
        # one live decoder, one new frame, the output layer onto the en-us model's 5126 senones with that speaker's adapter: latency
        dict(name="proj one frame to senones", op="proj", dtype="bf16", n_utt=1, frames=1, ragged=0, d_in=1024, d_out=5126, rank=16, n_adapters=8),
        # 512 live decoders, one new frame each, every speaker with an adapter: a hidden layer
        dict(name="proj 512 streams", op="proj", dtype="bf16", n_utt=512, frames=1, ragged=0, d_in=1024, d_out=1024, rank=16, n_adapters=128),
        # the first layer over a window of 11 frames of 39 features, in the features' own type, a ragged batch
        dict(name="proj first layer f32", op="proj", dtype="f32", n_utt=64, frames=600, ragged=1, d_in=429, d_out=1024, rank=8, n_adapters=24),
        # the output layer for a batch of whole utterances
        dict(name="proj batch to senones", op="proj", dtype="f16", n_utt=16, frames=2998, ragged=0, d_in=1024, d_out=5126, rank=24, n_adapters=16),
        # the largest: a hidden layer over 128 utterances of 30 s
        dict(name="proj large batch", op="proj", dtype="bf16", n_utt=128, frames=2998, ragged=0, d_in=1024, d_out=1024, rank=32, n_adapters=64),
        # one live decoder, one frame
        dict(name="norm one frame", op="norm", dtype="bf16", n_utt=1, frames=1, ragged=0, channels=1024, groups=32, act="silu"),
        # 512 live decoders, 100 ms each
        dict(name="norm 512 streams", op="norm", dtype="f16", n_utt=512, frames=10, ragged=0, channels=1024, groups=32, act="relu"),
        # a ragged batch of 1 to 30 s in the features' type, an odd number of channels a group
        dict(name="norm ragged f32", op="norm", dtype="f32", n_utt=64, frames=1600, ragged=1, channels=429, groups=11, act="silu"),
        # 128 utterances of 30 s
        dict(name="norm large batch", op="norm", dtype="bf16", n_utt=128, frames=2998, ragged=0, channels=1024, groups=32, act="gelu"),
        # one live decoder, one frame of 5126 senones
        dict(name="senones one frame", op="senones", dtype="f32", n_utt=1, frames=1, ragged=0, n_sen=5126),
        # 512 live decoders, 100 ms each
        dict(name="senones 512 streams", op="senones", dtype="f16", n_utt=512, frames=10, ragged=0, n_sen=5126),
        # 32 utterances of 30 s
        dict(name="senones batch", op="senones", dtype="bf16", n_utt=32, frames=2998, ragged=0, n_sen=5126),
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: streams of one frame up to batches of 30 s utterances, layers of 39 to 2048 inputs and 64 to 8192 outputs."""
    op = rng.choice(["proj", "norm", "senones"])
    c = dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), n_utt=_logint(rng, 1, 512), frames=_logint(rng, 1, 2998), ragged=rng.randint(0, 1))
    if op == "proj":
        c.update(d_in=_logint(rng, 39, 2048), d_out=_logint(rng, 64, 8192), rank=rng.randint(1, 64), n_adapters=_logint(rng, 1, 128))
        cost = lambda: (2.0 * c["n_utt"] * c["frames"] * c["d_in"] * c["d_out"] * (4 if c["dtype"] == "f32" else 1) > 7.0e11            # noqa: E731
                        or c["n_utt"] * c["frames"] * (c["d_in"] + c["d_out"]) > 6.0e8)
    elif op == "norm":
        groups = _logint(rng, 1, 64)
        c.update(groups=groups, channels=groups * _logint(rng, 1, max(1, 2048 // groups)), act=rng.choice(["none", "relu", "silu", "gelu"]))
        cost = lambda: c["n_utt"] * c["frames"] * c["channels"] > 3.5e8                                                                 # noqa: E731
    else:
        c.update(n_sen=_logint(rng, 100, 20000))
        cost = lambda: c["n_utt"] * c["frames"] * c["n_sen"] > 4.5e8                                                                    # noqa: E731
    while cost():                       # no dearer than the largest listed case: fewer utterances, then shorter ones
        if c["n_utt"] > 8:
            c["n_utt"] = c["n_utt"] * 2 // 3
        else:
            c["frames"] = c["frames"] * 2 // 3
    return c


def _lengths(case):
    """Frames per utterance: all alike, or spread between a fifteenth of the nominal length and as much short of twice it (the mean is the
    nominal one); the same for every seed, so that a case is one amount of work."""
    n, f = case["n_utt"], case["frames"]
    if not case["ragged"]:
        return [f] * n
    return [max(1, f // 15 + (2 * f - 2 * (f // 15)) * ((7919 * (u + 1)) % 1009) // 1009) for u in range(n)]


def _slots(case):
    """Which adapter each utterance has: speakers in no order, every eighth utterance without one."""
    return [-1 if u % 8 == 5 else (5 * u + u // 7) % case["n_adapters"] for u in range(case["n_utt"])]


def work(case):
    rows, es = sum(_lengths(case)), SIZES[case["dtype"]]
    if case["op"] == "proj":
        used = len(set(s for s in _slots(case) if s >= 0))
        with_adapter = sum(n for n, s in zip(_lengths(case), _slots(case)) if s >= 0)
        i, o, r = case["d_in"], case["d_out"], case["rank"]
        return {"bytes": es * (rows * (i + o) + i * o + used * r * (i + o)) + 4 * o, "flops": 2 * rows * i * o + 2 * with_adapter * r * (i + o)}
    if case["op"] == "norm":
        return {"bytes": 2 * rows * case["channels"] * es + 8 * case["channels"], "flops": 10 * rows * case["channels"]}
    return {"bytes": rows * case["n_sen"] * (es + 2) + 4 * (rows + case["n_sen"]), "flops": 9 * rows * case["n_sen"]}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, lens = DTYPES[case["dtype"]], _lengths(case)
    rows = sum(lens)

    def rand(*shape, scale=1.0, dtype=dt):
        out = torch.empty(shape, dtype=dtype, device="cuda")
        flat = out.view(-1)
        for i in range(0, flat.numel(), 1 << 27):           # in pieces: the 32-bit numbers of the largest inputs need not all live at once
            n = min(1 << 27, flat.numel() - i)
            flat[i:i + n] = (torch.randn(n, generator=g, device="cuda") * scale).to(dtype)
        return out

    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    s = dict(case=case, lens=lens, rows=rows, off=torch.tensor(off, dtype=torch.int32, device="cuda"))
    if case["op"] == "proj":
        i, o, r, na = case["d_in"], case["d_out"], case["rank"], case["n_adapters"]
        s.update(x=rand(rows, i), weight=rand(o, i, scale=i ** -0.5), bias=rand(o, scale=0.1, dtype=torch.float32),
                 a=rand(na, r, i, scale=i ** -0.5), b=rand(na, o, r, scale=0.3 * r ** -0.5), scale=2.0,
                 slots=_slots(case), slot_dev=torch.tensor(_slots(case), dtype=torch.int32, device="cuda"))
    elif case["op"] == "norm":
        c = case["channels"]
        # channels of unlike size and offset, as a layer's outputs are
        level = rand(c, scale=2.0, dtype=torch.float32)
        spread = torch.exp(rand(c, scale=0.5, dtype=torch.float32))
        x = rand(rows, c)
        for i in range(0, rows, 1 << 16):
            x[i:i + (1 << 16)] = (x[i:i + (1 << 16)].float() * spread + level).to(dt)
        s.update(x=x, weight=1.0 + rand(c, scale=0.2, dtype=torch.float32), bias=rand(c, scale=0.2, dtype=torch.float32), eps=1e-5)
    else:
        n = case["n_sen"]
        # outputs of a trained network: most senones far below the few that fit the frame; priors of a long-tailed senone count
        s.update(z=rand(rows, n, scale=4.0), prior=torch.log_softmax(rand(n, scale=1.0, dtype=torch.float32).double(), 0).float(), scale=0.8)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "proj":
        if own:
            from pocketsphinx_amd import AdaptedProjection
            s["layer"] = AdaptedProjection(s["weight"], s["bias"], max_adapters=case["n_adapters"], max_rank=case["rank"])
            for k in range(case["n_adapters"]):
                s["layer"].set_adapter(k, s["a"][k], s["b"][k], s["scale"])
        row = []                        # the adapter of every row, and each used adapter's rows: what a plain program keeps of its batch
        for n, k in zip(s["lens"], s["slots"]):
            row += [k] * n
        row = torch.tensor(row, dtype=torch.int64, device="cuda")
        s["row_slot"] = row
        s["rows_of"] = {k: torch.nonzero(row == k).view(-1) for k in sorted(set(s["slots"])) if k >= 0} if s["rows"] > 4096 else None
    elif case["op"] == "norm":
        s["utt_of_row"] = torch.repeat_interleave(torch.arange(case["n_utt"], device="cuda"), torch.tensor(s["lens"], device="cuda"))
        s["len_dev"] = torch.tensor(s["lens"], dtype=torch.float64, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------------------

def _activate(name, v):
    if name == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    return v


def run(state):
    case = state["case"]
    if case["op"] == "proj":
        return _proj_own(state) if own else _proj_plain(state)
    if case["op"] == "norm":
        return _norm_own(state) if own else _norm_plain(state)
    return _senones_own(state) if own else _senones_plain(state)


def _proj_own(s):
    return s["layer"](s["x"], utt_off=s["off"], adapter=s["slot_dev"])


def _proj_plain(s):
    x = s["x"].float()
    y = x @ s["weight"].float().t() + s["bias"]
    a, b = s["a"].float(), s["b"].float()
    na, r, _ = a.shape
    if s["rows_of"] is None:            # few rows: every adapter at once, the others' shares masked out
        h = (x @ a.reshape(na * r, -1).t()).view(-1, na, r)
        mine = s["row_slot"][:, None] == torch.arange(na, device=x.device)
        h = torch.where(mine[:, :, None], h, torch.zeros_like(h))
        y += s["scale"] * (h.view(-1, na * r) @ b.permute(0, 2, 1).reshape(na * r, -1))
    else:
        for k, rows in s["rows_of"].items():
            y[rows] += s["scale"] * ((x[rows] @ a[k].t()) @ b[k].t())
    return y.to(s["x"].dtype)


def _norm_own(s):
    from pocketsphinx_amd import group_norm
    c = s["case"]
    return group_norm(s["x"], s["off"], c["groups"], s["weight"], s["bias"], eps=s["eps"], act=c["act"])


def _sums_by_utterance(s, v):
    if s["case"]["n_utt"] <= 128:       # few utterances: one sum each; many: every row added to its utterance's
        return torch.stack([p.sum(0) for p in torch.split(v, s["lens"])])
    return torch.zeros((s["case"]["n_utt"], v.shape[1]), dtype=v.dtype, device=v.device).index_add(0, s["utt_of_row"], v)


def _norm_plain(s):
    c = s["case"]
    g, per = c["groups"], c["channels"] // c["groups"]
    x = s["x"].float().view(-1, g, per)
    count = (s["len_dev"] * per)[:, None]
    mean = _sums_by_utterance(s, x.sum(2, dtype=torch.float64)) / count
    d = x - mean[s["utt_of_row"]].float()[:, :, None]
    var = _sums_by_utterance(s, (d * d).sum(2, dtype=torch.float64)) / count
    d = d * (1.0 / torch.sqrt(var + s["eps"]))[s["utt_of_row"]].float()[:, :, None]
    y = _activate(c["act"], d.view(-1, c["channels"]) * s["weight"] + s["bias"])
    return y.to(s["x"].dtype)


def _senones_own(s):
    from pocketsphinx_amd import senone_scores
    return senone_scores(s["z"], s["prior"], scale=s["scale"], logbase=LOGBASE, want_best=True)


def _senones_plain(s):
    # in 64 bits: a score next to a rounding border is decided by the last bits of the difference
    unit = s["scale"] / (math.log(LOGBASE) * (1 << SENSCR_SHIFT))
    prior = s["prior"].double()
    scores = torch.empty(s["z"].shape, dtype=torch.int16, device=s["z"].device)
    best = torch.empty(s["rows"], dtype=torch.float32, device=s["z"].device)
    step = max(1, (1 << 27) // s["z"].shape[1])
    for i in range(0, s["rows"], step):
        z = s["z"][i:i + step].double()
        l = z - prior
        top = l.max(1, keepdim=True).values
        scores[i:i + step] = torch.clamp(torch.floor((top - l) * unit + 0.5), max=32767.0).to(torch.int16)
        zmax = z.max(1, keepdim=True).values
        best[i:i + step] = (top - (zmax + torch.log(torch.exp(z - zmax).sum(1, keepdim=True)))).view(-1).float()
    return scores, best


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    edges = [int(v) for v in s["off"].tolist()]
    if case["op"] == "proj":
        w, b = s["weight"].double(), s["bias"].double()
        y = torch.empty((s["rows"], case["d_out"]), dtype=torch.float64, device="cuda")
        for u, k in enumerate(s["slots"]):
            full = w if k < 0 else w + s["scale"] * torch.mm(s["b"][k].double(), s["a"][k].double())
            torch.addmm(b, s["x"][edges[u]:edges[u + 1]].double(), full.t(), out=y[edges[u]:edges[u + 1]])
        return y
    if case["op"] == "norm":
        y = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
        w, b = s["weight"].double(), s["bias"].double()
        for u in range(case["n_utt"]):
            x = s["x"][edges[u]:edges[u + 1]].double().reshape(edges[u + 1] - edges[u], case["groups"], -1)
            var, mean = torch.var_mean(x, dim=(0, 2), correction=0, keepdim=True)
            v = ((x - mean) / torch.sqrt(var + s["eps"])).reshape(x.shape[0], -1) * w + b
            if case["act"] == "relu":
                v = v.clamp(min=0.0)
            elif case["act"] == "silu":
                v = v * torch.sigmoid(v)
            elif case["act"] == "gelu":
                v = v * 0.5 * torch.erfc(-v / math.sqrt(2.0))
            y[edges[u]:edges[u + 1]] = v
        return y
    scores = torch.empty(s["z"].shape, dtype=torch.int16, device="cuda")
    best = torch.empty(s["rows"], dtype=torch.float64, device="cuda")
    nats = math.log(LOGBASE) * 2.0 ** SENSCR_SHIFT / s["scale"]
    for lo in range(0, s["rows"], 4096):
        z = s["z"][lo:lo + 4096].double()
        like = z - s["prior"].double()
        top = like.amax(1)
        scores[lo:lo + 4096] = ((top[:, None] - like) / nats + 0.5).floor().clamp(max=32767).to(torch.int16)
        best[lo:lo + 4096] = top - torch.logsumexp(z, 1)
    return scores, best
