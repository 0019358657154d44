"""Cases of the operators around a residual quantizer's training and decoding step: what each one is called with, its plain form in
torch, and its value in 64 bits.

* ``select``  -- `beam_select`: the best continuations over beams and codes (or any vocabulary), with the log-softmax of the scores and
  its gradient.
* ``reorder`` -- `beam_reorder`: the states of the beams follow the selection, with the gradient.
* ``norm``    -- `group_norm`: group norm with an activation on channels-last rows, forward and backward.
* ``clip``    -- `clip_grads`: the global norm of many gradients and the clipped gradients.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
WIDTH = {"fp32": 4, "bf16": 2, "fp16": 2}
NEG = float("-inf")


# ---------------------------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one stage of a residual quantizer's beam search: 8 x 1024 vectors, 4 beams with 4 codes each, scores are negative errors
        dict(name="select_residual_stage", op="select", batch=8192, beams=4, vocab=4, k=4, dtype="fp32", normalize=False,
             mask="none", finished=0.0, first=False, train=False),
        # decoding code tokens, 8 codebooks of 1024 codes flattened into one vocabulary: the mask admits the current stage's codes,
        # some beams have ended
        dict(name="select_stage_codes", op="select", batch=32, beams=5, vocab=8193, k=5, dtype="bf16", normalize=True,
             mask="stage", finished=0.2, first=False, train=False),
        # a large vocabulary, many beams: the widest rows, an odd length
        dict(name="select_wide_vocabulary", op="select", batch=16, beams=8, vocab=131071, k=8, dtype="bf16", normalize=True,
             mask="none", finished=0.0, first=False, train=False),
        # sequence-level training: the scores of the surviving beams are differentiated
        dict(name="select_train", op="select", batch=24, beams=4, vocab=32001, k=4, dtype="fp32", normalize=True,
             mask="none", finished=0.0, first=False, train=True),
        # the key and value caches of four layers follow their beams, a length that is no power of two
        dict(name="reorder_caches", op="reorder", batch=8, beams=5, k=5, train=False, kind="caches",
             dtype="bf16", layers=4, heads=8, length=777, width=64),
        # the states of a residual beam search with 8 quantizers at dim 256, in training
        dict(name="reorder_residual_states", op="reorder", batch=8192, beams=4, k=4, train=True, kind="residual",
             dtype="fp32", dim=256, stages=5),
        # one small map ahead of a quantizer at inference: latency
        dict(name="norm_one_map", op="norm", batch=1, rows=256, dim=512, groups=32, dtype="bf16", weight="fp32", activation="silu",
             padded=False, train=False),
        # the widest maps of an image decoder
        dict(name="norm_large_maps", op="norm", batch=6, rows=65536, dim=128, groups=32, dtype="bf16", weight="fp32",
             activation="silu", padded=False, train=False),
        # a training step at the quantizer's resolution and dim
        dict(name="norm_train", op="norm", batch=16, rows=1024, dim=256, groups=32, dtype="fp32", weight="fp32", activation="silu",
             padded=False, train=True),
        # a padded batch of audio frames in training, an odd length
        dict(name="norm_train_padded", op="norm", batch=8, rows=4099, dim=384, groups=8, dtype="bf16", weight="fp32",
             activation="none", padded=True, train=True),
        # the codebooks of a residual quantizer with 8 x 1024 codes at dim 256
        dict(name="clip_codebooks", op="clip", tensors=8, elements=8 * 1024 * 256, even=True, dtype="fp32", max_norm=1.0),
        # the gradients of a whole encoder and decoder: many tensors, from single biases to large weights
        dict(name="clip_model", op="clip", tensors=311, elements=90_000_000, even=False, dtype="mixed", max_norm=1.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["select", "select", "reorder", "norm", "norm", "clip"])
    if op == "select":
        if rng.random() < 0.3:
            beams, vocab = rng.randint(1, 8), rng.randint(1, 8)
            batch, norm, mask, fin, train = _log_int(rng, 1, 16384), False, "none", 0.0, rng.random() < 0.3
        else:
            beams, vocab = rng.randint(1, 12), _log_int(rng, 200, 131071)
            batch = _log_int(rng, 1, max(1, min(256, 16_000_000 // (beams * vocab))))
            norm, mask, train = True, rng.choice(["none", "none", "stage", "each"]), rng.random() < 0.3
            fin = rng.choice([0.0, 0.0, 0.3])
        if train:
            batch = max(1, batch // 3)
        first = norm and beams > 1 and fin == 0.0 and rng.random() < 0.2
        k = min(rng.randint(1, 16), beams * vocab if not (first or mask == "stage") else vocab // 8)
        return dict(op=op, batch=batch, beams=beams, vocab=vocab, k=k, dtype=rng.choice(["fp32", "bf16", "fp16"]), normalize=norm,
                    mask=mask, finished=fin, first=first, train=train)
    if op == "reorder":
        train = rng.random() < 0.4
        beams, k = rng.randint(1, 8), rng.randint(1, 8)
        if train or rng.random() < 0.3:
            dim = _log_int(rng, 8, 512)
            batch = _log_int(rng, 1, 8_000_000 // (8 * dim))
            stages = rng.randint(1, 8)
            return dict(op=op, batch=batch, beams=beams, k=k, train=train, kind="residual", dtype=rng.choice(["fp32", "bf16"]),
                        dim=dim, stages=stages)
        else:
            heads, length, width = rng.choice([1, 2, 4, 8]), _log_int(rng, 1, 2048), rng.choice([32, 64, 80, 128])
            layers = rng.randint(1, 8)
            batch = _log_int(rng, 1, max(1, min(32, 64_000_000 // (16 * heads * length * width * layers))))
            return dict(op=op, batch=batch, beams=beams, k=k, train=False, kind="caches", dtype=rng.choice(["bf16", "fp16"]),
                        layers=layers, heads=heads, length=length, width=width)
    if op == "norm":
        train = rng.random() < 0.5
        groups = rng.choice([1, 4, 8, 16, 32])
        dim = groups * rng.choice([1, 2, 3, 4, 8, 12, 16, 24, 32])
        while dim > 1024 or dim < 16:
            dim = groups * rng.choice([1, 2, 3, 4, 8, 12, 16, 24, 32])
        rows = _log_int(rng, -(-256 // (dim // groups)), 65536)
        batch = _log_int(rng, 1, max(1, min(32, (16_000_000 if train else 48_000_000) // (rows * dim))))
        dt = rng.choice(["fp32", "bf16", "fp16"])
        return dict(op=op, batch=batch, rows=rows, dim=dim, groups=groups, dtype=dt, weight=rng.choice(["fp32", dt]),
                    activation=rng.choice(["none", "silu"]), padded=rng.random() < 0.3, train=train)
    tensors = _log_int(rng, 1, 400)
    return dict(op=op, tensors=tensors, elements=_log_int(rng, 4 * tensors, 60_000_000), even=rng.random() < 0.3,
                dtype=rng.choice(["fp32", "bf16", "mixed"]), max_norm=rng.choice([1.0, 1.0, 0.1, 1e6]))


def _states(case):
    """(type, shape behind the beams) of every state that follows the beams"""
    if case["kind"] == "caches":                                    # keys and values of every layer
        return [(case["dtype"], (case["heads"], case["length"], case["width"]))] * (2 * case["layers"])
    # residual, sum of the codes, codes and losses of the stages so far
    return [(case["dtype"], (case["dim"],))] * 2 + [("int64", (case["stages"],)), ("fp32", (case["stages"],))]


def _clip_sizes(case):
    """elements of every tensor: all alike, or spread over many magnitudes as biases and weights are"""
    n, total = case["tensors"], case["elements"]
    if case["even"]:
        return [max(1, total // n)] * n
    r = random.Random(n * 7919 + total)
    w = [math.exp(r.uniform(0.0, 9.0)) for _ in range(n)]
    s = sum(w)
    return [max(1, int(total * v / s)) for v in w]


def _clip_dtype(case, i):
    return {"fp32": "fp32", "bf16": "bf16", "mixed": "fp32" if i % 3 == 0 else "bf16"}[case["dtype"]]


def _clip_places(case):
    """where every tensor begins in the bucket of its type (on a multiple of 64 elements), and the buckets' sizes"""
    places, totals = [], {}
    for i, n in enumerate(_clip_sizes(case)):
        dt = _clip_dtype(case, i)
        places.append(totals.get(dt, 0))
        totals[dt] = places[-1] + -(-n // 64) * 64
    return places, totals


def work(case):
    op = case["op"]
    if op == "select":
        rows, v, w = case["batch"] * case["beams"], case["vocab"], WIDTH[case["dtype"]]
        n = rows * v
        io = rows * 4 + case["batch"] * case["k"] * 20
        io += {"none": 0, "stage": v, "each": n}[case["mask"]]
        return dict(bytes=n * w * (2 if case["train"] else 1) + io,
                    flops=n * (5 if case["normalize"] else 1) * (2 if case["train"] else 1))
    if op == "reorder":
        per = sum(_state_bytes(s) for s in _states(case))
        b = case["batch"] * case["k"] * (2 * per + 8)
        f = 0
        if case["train"]:
            gr = sum(_state_bytes(s) for s in _states(case) if s[0] != "int64")
            b += case["batch"] * ((case["k"] + case["beams"]) * gr + case["k"] * 8)
            f = case["batch"] * case["k"] * gr // 4
        return dict(bytes=b, flops=f)
    if op == "norm":
        n, w = case["batch"] * case["rows"] * case["dim"], WIDTH[case["dtype"]]
        return dict(bytes=n * w * (4 if case["train"] else 2), flops=n * (28 if case["train"] else 10))
    sizes = _clip_sizes(case)
    return dict(bytes=sum(2 * s * WIDTH[_clip_dtype(case, i)] for i, s in enumerate(sizes)), flops=3 * sum(sizes))


def _state_bytes(s):
    return math.prod(s[1]) * {"int64": 8, **WIDTH}[s[0]]


# ---------------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1009 + 17)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    op = case["op"]
    st = dict(case=case)
    if op == "select":
        b, j, v, k = case["batch"], case["beams"], case["vocab"], case["k"]
        dt = DTYPES[case["dtype"]]
        if case["normalize"]:
            st["logits"] = (randn(b, j, v) * 2.0).to(dt)
        else:
            st["logits"] = (-0.05 * rand(b, j, v)).to(dt)            # negative mean squared errors of the codes
        scores = -torch.cumsum(rand(b, j), -1) * (0.3 if case["normalize"] else 0.02)
        if case["first"]:
            scores[:, 0], scores[:, 1:] = 0.0, NEG                   # the first token: one live beam
        st["scores"] = scores
        st["mask"] = None
        if case["mask"] == "stage":
            st["mask"] = torch.zeros(v, dtype=torch.bool, device="cuda")
            n = max(1, v // 8)
            st["mask"][2 * n:3 * n] = True
            st["mask"][v - 1] = True                                 # the end token
        elif case["mask"] == "each":
            st["mask"] = rand(b, j, v) < 0.5
        st["finished"] = (rand(b, j) < case["finished"]) if case["finished"] > 0 else None
        if case["train"]:
            st["logits"].requires_grad_(True)
            st["scores"].requires_grad_(True)
            st["grad"] = randn(b, k)
    elif op == "reorder":
        b, j, k = case["batch"], case["beams"], case["k"]
        st["states"] = []
        for dt, shape in _states(case):
            if dt == "int64":
                st["states"].append(torch.randint(0, 1024, (b, j, *shape), generator=g, device="cuda"))
            else:
                st["states"].append(randn(b, j, *shape).to(DTYPES[dt]))
        st["parents"] = torch.randint(0, j, (b, k), generator=g, device="cuda")
        if case["train"]:
            st["grads"] = [randn(b, k, *s.shape[2:]).to(s.dtype) for s in st["states"] if s.is_floating_point()]
            for s in st["states"]:
                if s.is_floating_point():
                    s.requires_grad_(True)
        else:
            st["out"] = [s.new_empty(b, k, *s.shape[2:]) for s in st["states"]]      # the other half of a double buffer
    elif op == "norm":
        b, n, c = case["batch"], case["rows"], case["dim"]
        dt, wt = DTYPES[case["dtype"]], DTYPES[case["weight"]]
        st["x"] = (randn(b, n, c) * (0.5 + rand(c)) + randn(c)).to(dt)
        st["weight"] = (1.0 + 0.2 * randn(c)).to(wt)
        st["bias"] = (0.2 * randn(c)).to(wt)
        st["lens"] = None
        if case["padded"]:
            st["lens"] = torch.randint(max(1, n // 4), n + 1, (b,), generator=g, device="cuda")
        if case["train"]:
            st["grad"] = randn(b, n, c).to(dt)
            for t in (st["x"], st["weight"], st["bias"]):
                t.requires_grad_(True)
    else:
        sizes = _clip_sizes(case)
        st["grads"] = [(0.01 * randn(s)).to(DTYPES[_clip_dtype(case, i)]) for i, s in enumerate(sizes)]
        # the clipped gradients go into one flat bucket of each type, as a data-parallel program keeps them
        places, totals = _clip_places(case)
        st["flat"] = {dt: torch.zeros(n, dtype=DTYPES[dt], device="cuda") for dt, n in totals.items()}
        st["out"] = [st["flat"][_clip_dtype(case, i)][at:at + n] for i, (at, n) in enumerate(zip(places, sizes))]
    return st


# ---------------------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _end(case):
    return case["vocab"] - 1


def _run_own(st):
    import vector_quantize_pytorch_amd as vq

    case = st["case"]
    op = case["op"]
    if op == "select":
        step = vq.beam_select(st["logits"], st["scores"], case["k"], mask=st["mask"], finished=st["finished"], end_token=_end(case),
                              normalize=case["normalize"])
        out = dict(scores=step.scores, parents=step.parents, tokens=step.tokens)
        if case["train"]:
            out["d_logits"], out["d_scores"] = torch.autograd.grad(step.scores, (st["logits"], st["scores"]), st["grad"])
        return out
    if op == "reorder":
        if not case["train"]:
            return vq.beam_reorder(st["states"], st["parents"], out=st["out"])
        new = vq.beam_reorder(st["states"], st["parents"])
        leaves = [s for s in st["states"] if s.requires_grad]
        return new + list(torch.autograd.grad([t for t in new if t.is_floating_point()], leaves, st["grads"]))
    if op == "norm":
        act = None if case["activation"] == "none" else case["activation"]
        y = vq.group_norm(st["x"], case["groups"], st["weight"], st["bias"], activation=act, lens=st["lens"])
        if not case["train"]:
            return y
        return [y, *torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["grad"])]
    _, norm = vq.clip_grads(st["grads"], case["max_norm"], out=st["out"])
    return dict(norm=norm, **st["flat"])


@torch.no_grad()
def _run_plain(st):
    return {"select": _plain_select, "reorder": _plain_reorder, "norm": _plain_norm, "clip": _plain_clip}[st["case"]["op"]](st)


def _plain_select(st):
    case = st["case"]
    k = case["k"]
    # (64 bits: the selection compares sums that may lie next to each other)
    x = st["logits"].double()
    b, j, v = x.shape
    if st["mask"] is not None:
        x = x.masked_fill(~st["mask"], NEG)
    prob = None
    if case["normalize"]:
        m = x.amax(-1, keepdim=True)
        e = (x - m).exp()
        z = e.sum(-1, keepdim=True)
        prob = e / z
        x = x - m - z.log()
    if st["finished"] is not None:
        only_end = torch.full((v,), NEG, dtype=torch.float64, device=x.device)
        only_end[_end(case)] = 0.0
        x = torch.where(st["finished"][..., None], only_end, x)
    total = st["scores"].double()[..., None] + x
    flat = torch.where(total.isnan(), NEG, total).reshape(b, j * v)
    # the k best, equal ones from the lowest index on
    kth = flat.topk(k, -1).values[:, -1:]
    above, equal = flat > kth, flat == kth
    keep = above | (equal & (equal.cumsum(-1) <= k - above.sum(-1, keepdim=True)))
    place = torch.arange(j * v, device=x.device)
    sel = torch.where(keep, place, j * v).topk(k, -1, largest=False, sorted=True).values
    best, order = flat.gather(1, sel).sort(dim=-1, descending=True, stable=True)
    sel = sel.gather(1, order)
    parents, tokens = sel // v, sel % v
    out = dict(scores=best.float(), parents=parents, tokens=tokens)
    if case["train"]:
        g = torch.where(best > NEG, st["grad"], 0.0).double()
        onto = torch.zeros(b, j, dtype=torch.float64, device=x.device).scatter_add_(1, parents, g)
        d = torch.zeros(b, j * v, dtype=torch.float64, device=x.device).scatter_add_(1, sel, g).view(b, j, v)
        if prob is not None:
            d = d - torch.where(prob.isnan(), 0.0, prob) * onto[..., None]
        if st["finished"] is not None:
            d = torch.where(st["finished"][..., None], 0.0, d)
        out["d_logits"], out["d_scores"] = d.to(st["logits"].dtype), onto.float()
    return out


def _plain_reorder(st):
    case, par = st["case"], st["parents"]
    b, k = par.shape
    at = torch.arange(b, device=par.device)[:, None]
    new = [s[at, par] for s in st["states"]]
    if not case["train"]:
        return new
    grads = []
    for s, g in zip([s for s in st["states"] if s.requires_grad], st["grads"]):
        d = torch.zeros(s.shape, dtype=torch.float32, device=s.device)
        d.index_put_((at.expand(b, k), par), g.float(), accumulate=True)
        grads.append(d.to(s.dtype))
    return new + grads


def _plain_norm(st):
    case = st["case"]
    x = st["x"].float()
    b, n, c = x.shape
    grp = case["groups"]
    w, bias = st["weight"].float(), st["bias"].float()
    live = torch.ones(b, n, 1, dtype=torch.bool, device=x.device)
    if st["lens"] is not None:
        live = torch.arange(n, device=x.device)[None, :, None] < st["lens"][:, None, None]
    cnt = (live.sum((1, 2)).float() * (c // grp))[:, None]                                       # [b, 1]

    def over_group(t):                                                                            # [b, n, c] -> sums [b, groups]
        return (t * live).view(b, n, grp, c // grp).sum((1, 3))

    def spread(t):                                                                                # [b, groups] -> [b, 1, c]
        return t.repeat_interleave(c // grp, -1)[:, None]

    mean = over_group(x) / cnt
    xc = x - spread(mean)
    rstd = 1.0 / torch.sqrt(over_group(xc * xc) / cnt + 1e-5)
    xh = xc * spread(rstd)
    z = xh * w + bias
    silu = case["activation"] == "silu"
    s = 1.0 / (1.0 + torch.exp(-z)) if silu else None
    y = (z * s if silu else z) * live
    if not case["train"]:
        return y.to(st["x"].dtype)
    dz = st["grad"].float() * live
    if silu:
        dz = dz * (s * (1.0 + z * (1.0 - s)))
    dw, db = (dz * xh).sum((0, 1)), dz.sum((0, 1))
    dn = dz * w
    dx = (dn - spread(over_group(dn) / cnt) - xh * spread(over_group(dn * xh) / cnt)) * spread(rstd) * live
    return [y.to(st["x"].dtype), dx.to(st["x"].dtype), dw.to(st["weight"].dtype), db.to(st["bias"].dtype)]


def _plain_clip(st):
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for t in st["grads"]:
        f = t.double()
        total = total + (f * f).sum()
    norm = total.sqrt()
    coef = (st["case"]["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    for t, o in zip(st["grads"], st["out"]):
        o.copy_(t.float() * coef)
    return dict(norm=norm.float(), **st["flat"])


# ---------------------------------------------------------------------------------------------------------------------------------
# the value in 64 bits, from the definitions, on the host
# ---------------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)

    def host(t):
        t = t.detach()
        return t.cpu().numpy() if t.dtype in (torch.bool, torch.int64) else t.cpu().to(torch.float64).numpy()

    def select_of(case, a):
        b, j, v, k = case["batch"], case["beams"], case["vocab"], case["k"]
        val, par, tok = np.empty((b, k)), np.empty((b, k), dtype=np.int64), np.empty((b, k), dtype=np.int64)
        train = case["train"]
        d_logits = np.zeros((b, j, v)) if train else None
        d_scores = np.zeros((b, j)) if train else None
        for i in range(b):
            table = np.full((j, v), NEG)
            soft = np.zeros((j, v))
            for r in range(j):
                if "finished" in a and a["finished"][i, r]:
                    table[r, _end(case)] = a["scores"][i, r]
                    continue
                row = a["logits"][i, r]
                allowed = np.ones(v, dtype=bool)
                if "mask" in a:
                    allowed = a["mask"] if a["mask"].ndim == 1 else a["mask"][i, r]
                live = row[allowed]
                if not live.size:
                    continue
                if case["normalize"]:
                    top = live.max()
                    p = np.exp(live - top)
                    mass = p.sum()
                    table[r, allowed] = a["scores"][i, r] + (live - top - math.log(mass))
                    soft[r, allowed] = p / mass
                else:
                    table[r, allowed] = a["scores"][i, r] + live
            f = table.reshape(-1)
            # everything that is at least the k-th largest, then by value and place
            bound = np.partition(f, f.size - k)[f.size - k]
            some = np.flatnonzero(f >= bound)
            some = some[np.lexsort((some, -f[some]))][:k]
            val[i], par[i], tok[i] = f[some], some // v, some % v
            if train:
                for n, at in enumerate(some):
                    r, t = at // v, at % v
                    if f[at] == NEG:
                        continue
                    w = a["grad"][i, n]
                    d_scores[i, r] += w
                    if not ("finished" in a and a["finished"][i, r]):
                        d_logits[i, r, t] += w
                        if case["normalize"]:
                            d_logits[i, r] -= w * soft[r]
        out = dict(scores=torch.from_numpy(val), parents=torch.from_numpy(par), tokens=torch.from_numpy(tok))
        if train:
            out["d_logits"], out["d_scores"] = torch.from_numpy(d_logits), torch.from_numpy(d_scores)
        return out

    def norm_of(case, a):
        b, n, c, grp = case["batch"], case["rows"], case["dim"], case["groups"]
        y, dx, dw, db = np.zeros((b, n, c)), np.zeros((b, n, c)), np.zeros(c), np.zeros(c)
        for i in range(b):
            m = int(a["lens"][i]) if "lens" in a else n
            for q in range(grp):
                cols = slice(q * (c // grp), (q + 1) * (c // grp))
                blk, w, bias = a["x"][i, :m, cols], a["weight"][cols], a["bias"][cols]
                inv = 1.0 / math.sqrt(blk.var() + 1e-5)
                xh = (blk - blk.mean()) * inv
                z = w * xh + bias
                slope = 1.0
                if case["activation"] == "silu":
                    sg = 1.0 / (1.0 + np.exp(-z))
                    y[i, :m, cols], slope = z * sg, sg + z * sg * (1.0 - sg)
                else:
                    y[i, :m, cols] = z
                if case["train"]:
                    dz = a["grad"][i, :m, cols] * slope
                    dw[cols] += (dz * xh).sum(0)
                    db[cols] += dz.sum(0)
                    dn = dz * w
                    dx[i, :m, cols] = inv * (dn - dn.mean() - xh * (dn * xh).mean())
        return [torch.from_numpy(t) for t in ((y, dx, dw, db) if case["train"] else (y,))]

    if case["op"] == "select":
        return select_of(case, {n: host(t) for n, t in st.items() if torch.is_tensor(t)})
    if case["op"] == "reorder":
        par = host(st["parents"])
        states = [host(s) for s in st["states"]]
        out = [np.stack([s[i, p] for i, p in enumerate(par)]) for s in states]
        if case["train"]:
            gs = iter(st["grads"])
            for s, t in zip(states, st["states"]):
                if t.is_floating_point():
                    g, d = host(next(gs)), np.zeros(s.shape)
                    rows = np.arange(len(par))
                    for i in range(par.shape[1]):
                        d[rows, par[:, i]] += g[:, i]
                    out.append(d)
        return [torch.from_numpy(t) for t in out]
    if case["op"] == "norm":
        if case["batch"] * case["rows"] * case["dim"] > 60_000_000:
            return None
        out = norm_of(case, {n: host(t) for n, t in st.items() if torch.is_tensor(t)})
        return out if case["train"] else out[0]
    gs = [host(t) for t in st["grads"]]
    norm = math.sqrt(math.fsum(float(np.dot(t, t)) for t in gs))
    coef = min(1.0, case["max_norm"] / (norm + 1e-6))
    places, totals = _clip_places(case)
    flat = {dt: torch.zeros(n, dtype=torch.float64) for dt, n in totals.items()}
    for i, (at, t) in enumerate(zip(places, gs)):
        flat[_clip_dtype(case, i)][at:at + t.size] = torch.from_numpy(t * coef)
    return dict(norm=torch.tensor(norm, dtype=torch.float64), **flat)
