"""group_norm and clip_grads / clip_grad_norm_ against plain 64-bit implementations, their refusals, and one training step that runs them
together with the beam search of a residual quantizer."""
import ctypes
import itertools

import pytest
import torch

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---- group norm -----------------------------------------------------------------------------------------------------------------------
def norm_ref(x, groups, w=None, b=None, eps=1e-5, act=None, live=None, grad=None):
    """x [b, n, c] on the host in 64 bits -> y (and dx, dw, db)"""
    x = x.detach().cpu().double()
    bs, n, c = x.shape
    w = torch.ones(c, dtype=torch.float64) if w is None else w.detach().cpu().double()
    b = torch.zeros(c, dtype=torch.float64) if b is None else b.detach().cpu().double()
    m = torch.ones(bs, n, 1, 1, dtype=torch.float64) if live is None else live.cpu().double()[..., None, None]
    cg = c // groups
    cnt = (m.sum((1, 2, 3), keepdim=True) * cg).clamp(min=1)

    def mean(t):                                                            # [bs, n, groups, cg] -> [bs, 1, groups, 1] over live rows
        return (t * m).sum((1, 3), keepdim=True) / cnt

    t = x.view(bs, n, groups, cg)
    t = t - mean(t)
    r = 1.0 / (mean(t * t) + eps).sqrt()
    xh = t * r
    w, b = w.view(groups, cg), b.view(groups, cg)
    z = xh * w + b
    s = torch.sigmoid(z)
    y = ((z * s if act else z) * m).view(bs, n, c)
    if grad is None:
        return y
    dz = grad.cpu().double().view(bs, n, groups, cg) * (s * (1 + z * (1 - s)) if act else 1.0) * m
    dn = dz * w
    dx = (r * (dn - mean(dn) - xh * mean(dn * xh)) * m).view(bs, n, c)
    return y, dx, (dz * xh).sum((0, 1)).view(c), dz.sum((0, 1)).view(c)


def norm_inputs(b, n, c, dtype, wtype, seed=0, offset=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(b, n, c, generator=g) * (0.5 + torch.rand(c, generator=g)) + offset * torch.randn(c, generator=g)).to(DT[dtype]).cuda()
    w = (1 + 0.3 * torch.randn(c, generator=g)).to(DT[wtype]).cuda()
    q = (0.3 * torch.randn(c, generator=g)).to(DT[wtype]).cuda()
    return x, w, q, torch.randn(b, n, c, generator=g).to(DT[dtype]).cuda()


def check_forward(y, want, dtype, xmax, rmax):
    """xh = (x - mean) rstd carries the mean's and rstd's 32-bit roundings (2^-23 of |x| rstd and 2^-22 of |xh|), the affine map and the
    activation 8 half steps; the result is rounded once"""
    tol = half_step(dtype) * want.abs() + 2.0 ** -20 * (1 + want.abs()) + 2.0 ** -22 * xmax * rmax * 2
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert ((y.detach().cpu().double() - want).abs() <= tol).all()


NORMS = [(1, 1, 1, 1), (2, 1, 64, 2), (1, 7, 6, 3), (3, 16, 32, 32), (2, 49, 96, 8), (2, 256, 512, 32), (1, 1000, 128, 32), (5, 33, 40, 1),
         (2, 4099, 24, 4), (1, 20000, 64, 16), (3, 301, 1025, 5), (1, 5, 8192, 64), (2, 300, 8192, 8192), (1, 70000, 8, 2), (70, 9, 16, 4), (2, 2048, 257, 257), (2, 16384, 128, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wtype", [("fp32", "fp32"), ("bf16", "fp32"), ("bf16", "bf16"), ("fp16", "fp16")])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("b,n,c,groups", NORMS)
def test_norm(dev, b, n, c, groups, act, dtype, wtype):
    import vector_quantize_pytorch_amd as A
    x, w, q, _ = norm_inputs(b, n, c, dtype, wtype)
    y = A.group_norm(x, groups, w, q, activation=act)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    # (a group of one value, or of nearly equal ones, has rstd up to eps^-1/2 = 317)
    check_forward(y, norm_ref(x, groups, w, q, act=act), x.dtype, x.abs().max().item(), 317.0 if n * c // groups < 64 else 4.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("b,n,c,groups", [(1, 16, 8, 2), (3, 49, 96, 8), (2, 256, 512, 32), (1, 4099, 24, 4), (2, 20000, 16, 4), (3, 301, 1025, 5), (40, 130, 64, 8), (1, 300, 8192, 8192), (600, 3, 32, 1), (2, 16384, 128, 32)])
def test_norm_gradient(dev, b, n, c, groups, act, dtype):
    """dx: rstd times three terms of at most |dz w| + mean + |xh| mean, each with 16 half steps of 2^-24 and the error of xh (2^-21 of
    1 + |x| rstd), rounded once; dw, db: n b terms, each with that error, summed in 32 bits or more (a pairwise or blocked sum: at most
    64 half steps of the sum of magnitudes)"""
    import vector_quantize_pytorch_amd as A
    x, w, q, grad = norm_inputs(b, n, c, dtype, "fp32", seed=1)
    for t in (x, w, q):
        t.requires_grad_(True)
    dx, dw, db = torch.autograd.grad(A.group_norm(x, groups, w, q, activation=act), (x, w, q), grad)
    _, rx, rw, rb = norm_ref(x, groups, w, q, act=act, grad=grad)
    gmax, wmax = grad.abs().max().item(), w.abs().max().item()
    unit = 2.0 ** -19 * gmax * 1.2 * max(wmax, 1.0) * 8                    # |xh| <= 8 here; silu' <= 1.1
    assert dx.dtype == x.dtype and ((dx.cpu().double() - rx).abs() <= half_step(x.dtype) * rx.abs() + 4 * unit + (2.0 ** -25 if dtype == "fp16" else 0)).all()
    absum = grad.abs().double().sum((0, 1)).cpu()
    for got, want in ((dw, rw), (db, rb)):
        assert got.dtype == torch.float32
        assert ((got.cpu().double() - want).abs() <= 2.0 ** -24 * want.abs() + absum * 1.2 * 8 * (2.0 ** -20 + 64 * 2.0 ** -24)).all()


@pytest.mark.gpu
def test_norm_gradient_against_differences(dev):
    """f = sum y grad along a direction with |u| <= 1 at h = 2^-6: a central difference is off by h^2/6 |f'''|, |f'''| <= 200 sum|grad| / 100
    on this data (unit variance, n c = 384 values), and by the 2^-21 of each y over h"""
    import vector_quantize_pytorch_amd as A
    x, w, q, grad = norm_inputs(2, 12, 32, "fp32", "fp32", seed=4)
    g = torch.Generator().manual_seed(9)
    u = [(torch.rand(t.shape, generator=g) * 2 - 1).cuda() for t in (x, w, q)]
    ts = [t.requires_grad_(True) for t in (x, w, q)]
    ds = torch.autograd.grad(A.group_norm(x, 4, w, q, activation="silu"), ts, grad)
    h = 2.0 ** -6
    lo, hi = (A.group_norm(*(lambda a, b, c: (a, 4, b, c))(*[(t + s * h * d).detach() for t, d in zip(ts, u)]), activation="silu") for s in (-1, 1))
    diff = ((hi.double() - lo.double()) * grad).sum().item() / (2 * h)
    have = sum((d.double() * e).sum().item() for d, e in zip(ds, u))
    assert abs(diff - have) <= grad.abs().sum().item() * (h * h / 6 * 2 + 2.0 ** -21 * 4 / h)


@pytest.mark.gpu
@pytest.mark.parametrize("n,c,groups", [(9, 16, 4), (257, 40, 8), (9001, 32, 2)])
@pytest.mark.parametrize("kind", ["lens", "mask"])
def test_norm_padded(dev, n, c, groups, kind):
    """padding holds NaN and infinities; an entry without live rows; lens beyond n and below 0; the gradients see live rows alone"""
    import vector_quantize_pytorch_amd as A
    b = 5
    x, w, q, grad = norm_inputs(b, n, c, "bf16", "fp32", seed=7)
    if kind == "lens":
        lens = torch.tensor([n, 0, n // 2, n + 100, -3], dtype=torch.int32 if n == 9 else torch.int64)
        live = torch.arange(n)[None] < lens[:, None]
        kw = dict(lens=lens.cuda())
    else:
        live = torch.rand(b, n, generator=torch.Generator().manual_seed(2)) < 0.5
        live[1] = False
        live[2] = False
        live[2, n - 1] = True
        kw = dict(mask=live.cuda())
    pad = ~live.cuda()[..., None]
    clean = x.clone()
    x = torch.where(pad, torch.tensor([float("nan"), float("inf")], device="cuda").repeat(c)[:c].bfloat16(), x)
    dirty = torch.where(pad, float("nan"), grad)
    for t in (x, w, q):
        t.requires_grad_(True)
    y = A.group_norm(x, groups, w, q, activation="silu", **kw)
    dx, dw, db = torch.autograd.grad(y, (x, w, q), dirty)
    ry, rx, rw, rb = norm_ref(clean, groups, w, q, act="silu", live=live, grad=grad)
    check_forward(y, ry, x.dtype, clean.abs().max().item(), 4.0 if n > 9 else 60.0)
    assert (y[~live.cuda()] == 0).all() and (dx[~live.cuda()] == 0).all()
    scale = 2.0 ** -16 * grad.abs().max().item() * (1.0 if n > 9 else 15.0)
    assert ((dx.cpu().double() - rx).abs() <= half_step(x.dtype) * rx.abs() + scale).all()
    absum = (grad.abs().double() * live.cuda()[..., None]).sum((0, 1)).cpu()
    for got, want in ((dw, rw), (db, rb)):
        assert ((got.cpu().double() - want).abs() <= absum * 12 * 2.0 ** -18 + 2.0 ** -20).all()


@pytest.mark.gpu
def test_norm_far_from_zero(dev):
    """a mean 4096 times the deviation: sums of squares about zero would keep nothing; x itself holds 2^-24 of 4096 = 2^-12 of a
    deviation, which both sides read alike, so the 32-bit mean is off by 2^-12 and each value by 2^-12 more"""
    import vector_quantize_pytorch_amd as A
    g = torch.Generator().manual_seed(3)
    for n, c, groups in ((64, 32, 4), (5000, 32, 4), (40000, 16, 1)):
        x = (4096 + torch.randn(2, n, c, generator=g)).cuda()
        y = A.group_norm(x, groups)
        assert ((y.cpu().double() - norm_ref(x, groups)).abs() <= 2.0 ** -10).all()
        x[:, 0] = 1e6                                                      # an outlier where a pivot might be taken
        x[:, 1:] -= 4096
        z = A.group_norm(x, groups)
        want = norm_ref(x, groups)
        assert ((z.cpu().double() - want).abs() <= 2.0 ** -20 * want.abs() + 2.0 ** -18).all()
    big = (torch.randn(1, 300, 8, generator=g) * 1e18).cuda()              # squares beyond 1e36, sums beyond 32 bits
    want = norm_ref(big, 2)
    assert ((A.group_norm(big, 2).cpu().double() - want).abs() <= 2.0 ** -19 * (1 + want.abs())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("n", [64, 20000])
@pytest.mark.parametrize("value", [1.0, 1000.0, 30000.0])
def test_norm_flat_far_from_zero(dev, value, n, act, dtype):
    """Groups of one value: its 64-bit mean is the value, a 32-bit number, so xh is 0 and the result the activated bias, whatever the value and the
    number of rows.  The activation takes 2^-21 of it (exp2 of a rounded argument, a reciprocal, two products), then one rounding.
    Nearly flat (one row a step up): xh carries the mean's rounding, 2^-24 |mean| rstd, and the roundings of rstd, 2^-20 of |xh| + |mean| rstd 2^-20 |xh|
    (the lanes' means are rounded like the whole mean is, so the variance is off by 2 |mean| 2^-24 a deviation)"""
    import vector_quantize_pytorch_amd as A
    b, c, groups = 2, 32, 4
    g = torch.Generator().manual_seed(n)
    w, q = (1 + 0.3 * torch.randn(c, generator=g)).cuda(), (0.3 * torch.randn(c, generator=g)).cuda()
    x = torch.full((b, n, c), value).to(DT[dtype])
    y = A.group_norm(x.cuda(), groups, w, q, activation=act).cpu().double()
    want = q.cpu().double().expand(b, n, c)
    want = want * torch.sigmoid(want) if act else want
    assert ((y - want).abs() <= (half_step(DT[dtype]) + 2.0 ** -21) * want.abs()).all()
    x[:, n // 3] = torch.nextafter(x[:, n // 3].float(), torch.tensor(torch.inf)) if dtype == "fp32" else x[:, n // 3] * (1 + 2 * half_step(DT[dtype]))
    want = norm_ref(x, groups, w, q, act=act)
    t = x.double().view(b, n, groups, c // groups)
    t = t - t.mean((1, 3), keepdim=True)
    r = 1.0 / ((t * t).mean((1, 3), keepdim=True) + 1e-5).sqrt()
    xh, off = (t * r).abs(), x.double().abs().max() * r
    err = ((off * 2.0 ** -24 + xh * 2.0 ** -20 * (1 + off)).expand_as(t) * w.cpu().double().abs().view(groups, -1)).reshape(b, n, c)
    y = A.group_norm(x.cuda(), groups, w, q, activation=act).cpu().double()
    assert ((y - want).abs() <= half_step(DT[dtype]) * want.abs() + 1.1 * err * (1 + half_step(DT[dtype])) + 2.0 ** -21 * (want.abs() + err) + (2.0 ** -25 if dtype == "fp16" else 0)).all()


@pytest.mark.gpu
def test_norm_layouts_and_module(dev):
    import vector_quantize_pytorch_amd as A
    torch.manual_seed(0)
    norm = A.GroupNorm(8, 64, activation="silu", accept_image_fmap=True).cuda()
    torch.nn.init.normal_(norm.weight)
    plain = torch.nn.GroupNorm(8, 64).cuda()
    plain.load_state_dict(norm.state_dict())
    img = torch.randn(2, 64, 9, 13, device="cuda")
    want = torch.nn.functional.silu(torch.nn.functional.group_norm(img.cpu().double(), 8, plain.weight.cpu().double(), plain.bias.cpu().double()))
    for x in (img, img.contiguous(memory_format=torch.channels_last)):
        y = norm(x)
        assert y.is_contiguous(memory_format=torch.channels_last)
        assert ((y.cpu().double() - want).abs() <= 2.0 ** -18 * (1 + want.abs())).all()
    # a channels-last map goes on to a quantizer in place: its rows are the norm's rows
    rows = norm(img).flatten(2).transpose(1, 2)
    assert rows.is_contiguous()
    seq = A.GroupNorm(8, 64, channel_last=False, affine=False).cuda()(img.flatten(2))
    assert seq.shape == (2, 64, 117) and torch.allclose(seq, torch.nn.functional.group_norm(img, 8).flatten(2), atol=1e-4)
    wide = torch.randn(3, 2, 50, 96, device="cuda")
    for x in (wide[..., 8:72], wide[:, 1], wide[:, :, 1:40:3, :32], wide[0, 0], wide.transpose(1, 2), wide.transpose(0, 2)[..., ::2]):
        ref = norm_ref(x.reshape(x.shape[0], -1, x.shape[-1]) if x.ndim > 2 else x[:, None], 8).view(x.shape)
        assert ((A.group_norm(x, 8).cpu().double() - ref).abs() <= 2.0 ** -14 * (1 + ref.abs())).all()
    assert A.group_norm(torch.empty(0, 5, 16, device="cuda"), 4).shape == (0, 5, 16)
    empty = torch.empty(2, 0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y = A.group_norm(empty, 4, w)
    assert y.shape == (2, 0, 16)
    dx, dw = torch.autograd.grad(y, (empty, w), torch.empty(2, 0, 16, device="cuda"))
    assert dx.shape == (2, 0, 16) and (dw == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [64, 3000, 30000])
def test_norm_in_a_graph_and_repeatable(dev, n):
    """forward and backward captured twice (two graphs, workspaces apart), replayed in turn with eager work between; the sums have one order"""
    import vector_quantize_pytorch_amd as A
    sets = [norm_inputs(2, n, 64, "bf16", "fp32", seed=s) for s in (1, 2)]

    def step(x, w, q, grad):
        ts = [t.detach().requires_grad_(True) for t in (x, w, q)]
        y = A.group_norm(ts[0], 8, ts[1], ts[2], activation="silu")
        return (y, *torch.autograd.grad(y, ts, grad))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*sets[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*s))
        graphs.append(g)
    for r in range(3):
        for i, (g, o) in enumerate(zip(graphs, outs)):
            sets[i][0].copy_(norm_inputs(2, n, 64, "bf16", "fp32", seed=10 * r + i)[0])
            g.replay()
            eager = step(*sets[i])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(o, eager))


# ---- gradients ------------------------------------------------------------------------------------------------------------------------
def clip_ref(grads, max_norm):
    n = sum((g.cpu().double() ** 2).sum() for g in grads).sqrt()
    return n, min(1.0, float(max_norm / (n + 1e-6)))


def grads_of(sizes, types, scale=0.1, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(DT[types[i % len(types)]]).cuda() for i, s in enumerate(sizes)]


@pytest.mark.gpu
@pytest.mark.parametrize("types", [("fp32",), ("bf16",), ("fp16", "fp32", "bf16")])
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9])
@pytest.mark.parametrize("sizes", [(1,), (0,), (5, 0, 7), (16384, 16385, 16383), (1_000_003,), tuple(range(1, 330)), (4096,) * 101])
def test_clip(dev, sizes, max_norm, types):
    """norm: squares and sums in 64 bits, rounded to fp32 once; the factor is rounded once, the product once"""
    import vector_quantize_pytorch_amd as A
    grads = grads_of(sizes, types)
    n, coef = clip_ref(grads, max_norm)
    keep = [g.clone() for g in grads]
    out, norm = A.clip_grads(grads, max_norm)
    assert all(torch.equal(g, k) for g, k in zip(grads, keep))
    assert norm.shape == () and norm.dtype == torch.float32 and abs(norm.item() - n) <= 2.0 ** -23 * n
    inplace, again = A.clip_grads(grads, max_norm, out=grads)
    assert torch.equal(norm, again) and all(torch.equal(a, b) for a, b in zip(inplace, out))
    for o, k in zip(out, keep):
        want = k.cpu().double() * coef
        tiny = 2.0 ** -25 if k.dtype == torch.float16 else 0.0
        assert o.dtype == k.dtype and ((o.cpu().double() - want).abs() <= want.abs() * (half_step(k.dtype) * (1 + 2.0 ** -8) + 2.0 ** -22) + tiny).all()


@pytest.mark.gpu
def test_clip_extremes(dev):
    import vector_quantize_pytorch_amd as A
    for scale in (1e30, 1e-30):                                            # squares beyond 32 bits on either side
        g = torch.full((1000,), scale, device="cuda")
        (out,), norm = A.clip_grads([g], 1.0)
        assert abs(norm.item() / (scale * 1000 ** 0.5) - 1) < 1e-6
        assert torch.allclose(out, g / norm if scale > 1 else g, rtol=1e-6, atol=0.0)
    g = torch.ones(10, device="cuda")
    (out,), norm = A.clip_grads([torch.tensor([float("inf"), 1.0], device="cuda")], 1.0)
    assert norm.item() == float("inf") and out[1].item() == 0.0 and out[0].isnan()
    outs, norm = A.clip_grads([torch.tensor([float("nan")], device="cuda"), g], 1.0)
    assert norm.isnan() and outs[1].isnan().all()
    (out,), norm = A.clip_grads([g], float("inf"))                         # max_norm inf: the norm alone
    assert torch.equal(out, g) and abs(norm.item() - 10 ** 0.5) < 1e-6
    (out,), norm = A.clip_grads([torch.tensor([float("inf"), 2.0], device="cuda")], float("inf"))
    assert norm.item() == float("inf") and out.tolist() == [float("inf"), 2.0]
    assert A.clip_grads([], 1.0)[0] == []
    zero = [torch.zeros(5, device="cuda")]
    assert A.clip_grads(zero, 1.0)[1].item() == 0.0 and (A.clip_grads(zero, 1.0)[0][0] == 0).all()
    with torch.inference_mode():
        t = torch.ones(8, device="cuda")
        A.clip_grads([t], 1.0, out=[t])
        assert abs(t.norm().item() - 1) < 1e-5
    from vector_quantize_pytorch_amd._lib import VQHipError               # overlaps are refused before anything is launched
    t = torch.ones(32, device="cuda")
    for gs, out in (([t, t], None), ([t[:8]], [t[4:12]]), ([t[:16], t[20:24]], [t[:16], t[:4]]), ([t[:8], t[4:12]], [t[:8], t[4:12]])):
        with pytest.raises(VQHipError, match="twice|shares memory"):
            A.clip_grads(gs, 1.0, out=out)
    assert (t == 1).all()
    odd = torch.ones(4099, device="cuda", dtype=torch.bfloat16)            # addresses off every vector's alignment
    parts = [odd[1:8], odd[9:1000], odd[1001:4098]]
    A.clip_grads(parts, 1.0, out=parts)
    want = torch.tensor(1 / (sum(p.numel() for p in parts) ** 0.5 + 1e-6)).bfloat16()
    assert odd[0] == 1 and odd[8] == 1 and odd[1000] == 1 and odd[4098] == 1 and all((p == want.cuda()).all() for p in parts)


@pytest.mark.gpu
def test_clip_parameters(dev):
    """like torch.nn.utils.clip_grad_norm_: shared and missing gradients, a transposed one, the error on request (nothing is changed then)"""
    import vector_quantize_pytorch_amd as A
    a, b, c, d = (torch.nn.Parameter(torch.randn(33, 17, device="cuda")) for _ in range(4))
    a.grad, b.grad = torch.randn(33, 17, device="cuda"), torch.randn(17, 33, device="cuda").t()
    d.grad = a.grad
    ref = [p.grad.clone() for p in (a, b)]
    n = sum((r.double() ** 2).sum() for r in ref).sqrt()
    norm = A.clip_grad_norm_([a, b, c, d], 0.25)
    assert abs(norm.item() - n.item()) <= 2.0 ** -23 * n and c.grad is None and d.grad is a.grad
    for p, r in zip((a, b), ref):
        assert torch.allclose(p.grad.double(), r.double() * 0.25 / (n + 1e-6), rtol=2.0 ** -21, atol=0.0)
    assert A.clip_grad_norm_(iter([c]), 1.0).item() == 0.0
    assert abs(A.clip_grad_norm_(a, 1e9).item() - a.grad.double().norm().item()) < 1e-6
    a.grad[0, 0] = float("inf")
    before = [p.grad.clone() for p in (a, b)]
    with pytest.raises(RuntimeError, match="not finite"):
        A.clip_grad_norm_([a, b], 0.1, error_if_nonfinite=True)
    assert all(torch.equal(p.grad, r) for p, r in zip((a, b), before))
    # a graph that saved a clipped tensor notices
    t = torch.ones(4, device="cuda")
    s = (torch.ones(4, device="cuda", requires_grad=True) * t).sum()
    A.clip_grads([t], 0.5, out=[t])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        s.backward()


@pytest.mark.gpu
def test_clip_in_a_graph(dev):
    import vector_quantize_pytorch_amd as A
    grads = grads_of((70000, 3, 555) * 50, ("fp32", "bf16"))
    fresh = [grads_of((70000, 3, 555) * 50, ("fp32", "bf16"), seed=s) for s in range(3)]
    out = [torch.empty_like(g) for g in grads]
    A.clip_grads(grads, 1.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, norm = A.clip_grads(grads, 1.0, out=out)
    for f in fresh:
        for g, t in zip(grads, f):
            g.copy_(t)
        graph.replay()
        want, n = A.clip_grads(f, 1.0)
        torch.cuda.synchronize()
        assert torch.equal(n, norm) and all(torch.equal(o, w) for o, w in zip(out, want))


@pytest.mark.gpu
def test_in_place_codebook_optimizer_clips(dev):
    """VectorQuantize(in_place_codebook_max_grad_norm=): SGD moves the codebook by lr times the clipped gradient; a bound that is not
    reached changes nothing"""
    import vector_quantize_pytorch_amd as A
    from functools import partial
    torch.manual_seed(0)
    kw = dict(dim=32, codebook_size=64, learnable_codebook=True, ema_update=False, in_place_codebook_optimizer=partial(torch.optim.SGD, lr=1.0))
    vqs = [A.VectorQuantize(**kw, in_place_codebook_max_grad_norm=m).cuda().train() for m in (None, 1e6, 1e-3)]
    for v in vqs[1:]:
        v.load_state_dict(vqs[0].state_dict())
    before = vqs[0].codebook.detach().clone()
    x = torch.randn(2, 128, 32, device="cuda")
    for v in vqs:
        v(x)
    moved = [before - v.codebook.detach() for v in vqs]
    # a code's gradient adds 2 (code - row) / 8192 over its m rows by atomics, in any order: two runs differ by at most m steps of 2^-24 of the
    # m magnitudes each, and by the step's and the difference's roundings of the codebook (2 steps each)
    m = torch.cdist(x.flatten(0, 1), before).argmin(-1).bincount(minlength=64).float()[:, None]
    tol = 2.0 ** -24 * (2 * m * m * 2 * (x.abs().max() + before.abs().max()) / 8192 + 4 * before.abs())
    assert ((moved[0] - moved[1]).abs() <= tol).all() and moved[0].norm() > 1e-3
    assert abs(moved[2].norm().item() - 1e-3) < 2e-5
    cos = (moved[2] * moved[0]).sum() / (moved[2].norm() * moved[0].norm())
    assert cos > 1 - 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_training_step_of_a_tokenizer(dev, dtype):
    """the operators as they are used together: norm ahead of a residual quantizer with beams, loss, backward, clipping, optimizer step"""
    import vector_quantize_pytorch_amd as A
    torch.manual_seed(0)
    b, n, c = 2, 120, 64
    enc, dec = torch.nn.Linear(c, c).cuda().to(DT[dtype]), torch.nn.Linear(c, c).cuda().to(DT[dtype])
    norm = A.GroupNorm(8, c, activation="silu").cuda()
    rvq = A.ResidualVQ(dim=c, num_quantizers=4, codebook_size=128, beam_size=4).cuda().train()
    params = [*enc.parameters(), *norm.parameters(), *dec.parameters()]
    opt = torch.optim.SGD(params, lr=0.1)
    x = torch.randn(b, n, c, device="cuda").to(DT[dtype])
    lens = torch.tensor([n, n // 3], device="cuda")
    for _ in range(2):
        h = norm(enc(x), lens=lens)
        books = rvq.codebooks.clone()                       # (the forward moves the first one after its search)
        q, idx, commit = rvq(h)
        loss = (dec(q) - x).float().square().mean() + commit.sum()
        opt.zero_grad()
        loss.backward()
        ref = [p.grad.detach().clone() for p in params]
        total, coef = clip_ref(ref, 0.05)
        got = A.clip_grad_norm_(params, 0.05)
        assert abs(got.item() - total) <= 2.0 ** -23 * total
        for p, r in zip(params, ref):
            assert r.abs().sum() > 0 and ((p.grad.cpu().double() - r.cpu().double() * coef).abs() <= r.cpu().double().abs() * (half_step(r.dtype) * 1.01 + 2.0 ** -22)).all()
        before = [p.detach().clone() for p in params]
        opt.step()
        assert any(not torch.equal(p, t) for p, t in zip(params, before))
        assert idx.shape == (b, n, 4) and (idx >= 0).all() and torch.isfinite(q.float()).all()
        # the output is the sum of the codes that the indices name, each routed (a rotation of the row onto its code: 10 roundings in
        # the rows' type of values of at most the code's norm) and added in the rows' type; a zero row, padding, has no direction to rotate
        codes = torch.stack([books[i][idx[..., i]] for i in range(4)])
        tol = half_step(DT[dtype]) * 12 * codes.double().norm(dim=-1).sum(0)[..., None]
        far = (q.detach().double() - codes.double().sum(0)).abs() - tol
        assert far[torch.arange(n, device="cuda")[None] < lens[:, None]].max().item() <= 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("n,c,groups", [(9, 16, 4), (20000, 16, 4), (5, 1, 1)])
def test_norm_of_negated_tensors(dev, n, c, groups):
    """torch leaves a negation (the imaginary part of a conjugate, say) pending in a flag: rows, parameters and gradients count with it"""
    import vector_quantize_pytorch_amd as A
    ts = norm_inputs(2, n, c, "fp32", "fp32")

    def step(x, w, q, grad):
        x, w, q = (t.detach().requires_grad_(True) for t in (x, w, q))
        y = A.group_norm(x, groups, w, q, activation="silu")
        return (y, *torch.autograd.grad(y, (x, w, q), grad))

    want = step(*ts)
    for i in range(4):
        for flagged in (torch._neg_view(-ts[i]), torch.complex(ts[i], -ts[i]).conj().imag):
            assert flagged.is_neg() and all(torch.equal(a, b) for a, b in zip(step(*ts[:i], flagged, *ts[i + 1:]), want))


@pytest.mark.gpu
def test_clip_of_negated_tensors(dev):
    import vector_quantize_pytorch_amd as A
    from vector_quantize_pytorch_amd._lib import VQHipError
    g = torch.complex(*[torch.full((1,), 3.0, device="cuda")] * 2).conj().imag       # -3, contiguous, memory of +3
    h = torch.full((1,), 4.0, device="cuda")
    (a, b), norm = A.clip_grads([g, h], 2.5)
    assert norm.item() == 5.0 and abs(a.item() + 1.5) < 1e-6 and abs(b.item() - 2.0) < 1e-6
    o = [torch.empty(1, device="cuda") for _ in range(2)]
    A.clip_grads([g, h], 2.5, out=o)
    assert abs(o[0].item() + 1.5) < 1e-6 and abs(o[1].item() - 2.0) < 1e-6
    p = torch.nn.Parameter(torch.zeros(1, device="cuda"))
    p.grad = g
    A.clip_grad_norm_([p], 1.5)
    assert abs(p.grad.item() + 1.5) < 1e-6
    with pytest.raises(VQHipError, match="pending"):
        A.clip_grads([h], 1.0, out=[torch.complex(h, h).conj().imag])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("b,n,c,groups", [(2100, 2, 256, 32), (2100, 2, 64, 8), (2100, 3, 96, 4), (300, 16, 256, 8), (5, 3000, 64, 8), (20, 1024, 128, 32), (60, 256, 128, 32), (4, 8192, 32, 8)])
def test_norm_many_maps(dev, b, n, c, groups, dtype):
    """batches on either side of where one launch gives way to two"""
    import vector_quantize_pytorch_amd as A
    x, w, q, _ = norm_inputs(b, n, c, dtype, "fp32", seed=n)
    y = A.group_norm(x, groups, w, q, activation="silu")
    check_forward(y, norm_ref(x, groups, w, q, act="silu"), x.dtype, x.abs().max().item(), 317.0 if n * c // groups < 64 else 4.0)


# ---- refusals (host side: no GPU) -------------------------------------------------------------------------------------------------------
def test_norm_refusals():
    import vector_quantize_pytorch_amd as A
    from vector_quantize_pytorch_amd._lib import VQHipError
    x, w = torch.zeros(2, 5, 16), torch.ones(16)
    for match, call in [
            ("no CPU fallback", lambda: A.group_norm(x, 4)),
            ("no CPU fallback", lambda: A.GroupNorm(4, 16)(x)),
            ("unsupported dtype", lambda: A.group_norm(x.double(), 4)),
            ("expected", lambda: A.group_norm(torch.zeros(16), 4)),
            ("groups", lambda: A.group_norm(x, 3)),
            ("groups", lambda: A.group_norm(x, 0)),
            ("groups", lambda: A.group_norm(torch.zeros(1, 1, 8193), 1)),
            ("groups", lambda: A.GroupNorm(3, 16)),
            ("activation", lambda: A.group_norm(x, 4, activation="relu")),
            ("activation", lambda: A.GroupNorm(4, 16, activation="gelu")),
            ("eps", lambda: A.group_norm(x, 4, eps=-1.0)),
            ("eps", lambda: A.group_norm(x, 4, eps=float("nan"))),
            ("parameter", lambda: A.group_norm(x, 4, w[:8])),
            ("parameter", lambda: A.group_norm(x, 4, w.bfloat16())),
            ("weight of", lambda: A.group_norm(x.bfloat16(), 4, w, w.bfloat16())),
            ("mask and lens", lambda: A.group_norm(x, 4, mask=torch.ones(2, 5, dtype=torch.bool), lens=torch.ones(2, dtype=torch.int64))),
            ("mask", lambda: A.group_norm(x, 4, mask=torch.ones(2, 5))),
            ("mask", lambda: A.group_norm(x, 4, mask=torch.ones(5, dtype=torch.bool))),
            ("mask", lambda: A.group_norm(x[:, :, None], 4, mask=torch.ones(2, 5, dtype=torch.bool))),
            ("lens", lambda: A.group_norm(x, 4, lens=torch.ones(2))),
            ("lens", lambda: A.group_norm(x, 4, lens=torch.ones(3, dtype=torch.int64))),
            ("expected", lambda: A.GroupNorm(4, 16, accept_image_fmap=True)(x))]:
        with pytest.raises(VQHipError, match=match):
            call()


def test_clip_refusals():
    import vector_quantize_pytorch_amd as A
    from vector_quantize_pytorch_amd._lib import VQHipError
    g, h = torch.zeros(16), torch.zeros(4, 4)
    for match, call in [
            ("no CPU fallback", lambda: A.clip_grads([g], 1.0)),
            ("no CPU fallback", lambda: A.clip_grads([g], 1.0, out=[g])),
            ("max_norm", lambda: A.clip_grads([g], -1.0)),
            ("max_norm", lambda: A.clip_grads([g], float("nan"))),
            ("unsupported dtype", lambda: A.clip_grads([g.double()], 1.0)),
            ("contiguous", lambda: A.clip_grads([h.t()], 1.0)),
            ("results", lambda: A.clip_grads([g], 1.0, out=[])),
            ("out", lambda: A.clip_grads([g], 1.0, out=[g.half()])),
            ("out", lambda: A.clip_grads([g], 1.0, out=[h[:2]])),
            ("out", lambda: A.clip_grads([g], 1.0, out=[h.t()]))]:
        with pytest.raises(VQHipError, match=match):
            call()
    with pytest.raises(AssertionError):
        A.VectorQuantize(dim=8, codebook_size=8, in_place_codebook_max_grad_norm=1.0)


def test_c_entry_refusals():
    from vector_quantize_pytorch_amd import _lib
    from vector_quantize_pytorch_amd.grads import _Grad
    from vector_quantize_pytorch_amd.norms import _Norm
    L = _lib.lib()
    nws = L.vqhip_group_norm_workspace_bytes(2, 5, 16, 4)
    ok = dict(x=8, dtype=0, B=2, N=5, C=16, stride_b=80, stride_n=16, groups=4, param_dtype=0, eps=1e-5, mean=8, rstd=8, workspace=16, workspace_bytes=nws)
    for rc, change in [(-1, dict(dtype=3)), (-1, dict(param_dtype=-1)), (-1, dict(B=-1)), (-1, dict(C=0)), (-1, dict(groups=3)), (-1, dict(groups=0)), (-1, dict(eps=-1.0)),
                       (-1, dict(eps=float("nan"))), (-1, dict(activation=2)), (-2, dict(C=8196)), (-2, dict(N=2 ** 40)), (-2, dict(B=2 ** 31)), (-1, dict(lens=8, mask=8)),
                       (-1, dict(x=0)), (-1, dict(mean=0)), (-1, dict(workspace_bytes=nws - 1)), (-1, dict(workspace=0)), (0, dict(B=0)), (0, dict(N=0))]:
        s = _Norm(**{**ok, **change})
        assert L.vqhip_group_norm(ctypes.byref(s), 8, None) == rc, change
    s = _Norm(**{**ok, "workspace": 24})
    assert L.vqhip_group_norm(ctypes.byref(s), 8, None) == -3
    s = _Norm(**ok)
    assert L.vqhip_group_norm(ctypes.byref(s), None, None) == -1
    assert L.vqhip_group_norm_bwd(ctypes.byref(s), None, 8, 8, 8, None) == -1
    assert L.vqhip_group_norm_bwd(ctypes.byref(s), 8, None, None, None, None) == 0
    assert L.vqhip_group_norm(None, 8, None) == -1
    one = (_Grad * 1)((8, 8, 4, 0))
    assert L.vqhip_clip_grads(one, 1, 1.0, 1e-6, 8, 24, 64, None) == -3
    ws = L.vqhip_clip_grads_workspace_bytes(one, 1)
    for args in [(one, -1, 1.0, 1e-6, 8, 16, ws), (None, 1, 1.0, 1e-6, 8, 16, ws), (one, 1, -1.0, 1e-6, 8, 16, ws), (one, 1, float("nan"), 1e-6, 8, 16, ws),
                 (one, 1, 1.0, -1.0, 8, 16, ws), (one, 1, 1.0, 1e-6, None, 16, ws), (one, 1, 1.0, 1e-6, 8, None, ws), (one, 1, 1.0, 1e-6, 8, 16, ws - 1),
                 ((_Grad * 1)((8, 8, 4, 3)), 1, 1.0, 1e-6, 8, 16, ws), ((_Grad * 1)((8, 8, -4, 0)), 1, 1.0, 1e-6, 8, 16, ws),
                 ((_Grad * 1)((None, 8, 4, 0)), 1, 1.0, 1e-6, 8, 16, ws)]:
        assert L.vqhip_clip_grads(*args, None) == -1
    # overlaps: (src, dst, elements, fp32), bytes 4 a piece
    many = L.vqhip_clip_grads_workspace_bytes((_Grad * 2)((8, 8, 4, 0), (8, 8, 4, 0)), 2)
    for pair in [((64, 64, 4, 0), (64, 64, 4, 0)), ((64, None, 4, 0), (64, None, 4, 0)), ((64, 72, 4, 0), (256, 256, 4, 0)), ((64, 64, 4, 0), (76, 256, 4, 0)),
                 ((64, 128, 4, 0), (256, 140, 4, 0)), ((64, 128, 8, 0), (140, 256, 4, 0)), ((64, 64, 8, 0), (95, 95, 4, 0))]:
        args = ((_Grad * 2)(*pair), 2, 1.0, 1e-6, 8, 16, many)
        assert L.vqhip_clip_grads(*args, None) == -1


def test_forward_mode_is_refused():
    """a dual tensor's tangent would be lost: no entry point has a forward-mode derivative (host side: no GPU)"""
    import torch.autograd.forward_ad as fwad
    import vector_quantize_pytorch_amd as A
    from vector_quantize_pytorch_amd._lib import VQHipError
    x, w = torch.zeros(2, 5, 16), torch.ones(16)
    with fwad.dual_level():
        def dual(t):
            return fwad.make_dual(t, torch.ones_like(t))
        p = torch.nn.Parameter(torch.zeros(4))
        p.grad = dual(torch.ones(4))
        for call in (lambda: A.group_norm(dual(x), 4), lambda: A.group_norm(x, 4, dual(w)), lambda: A.group_norm(x, 4, w, dual(w)),
                     lambda: A.GroupNorm(4, 16)(dual(x)), lambda: A.clip_grads([x, dual(x)], 1.0), lambda: A.clip_grads([x], 1.0, out=[dual(x.clone())]),
                     lambda: A.clip_grad_norm_([p], 1.0)):
            with pytest.raises(VQHipError, match="forward-mode"):
                call()
        with pytest.raises(VQHipError, match="no CPU fallback"):             # a level without a tangent is no hindrance
            A.group_norm(x, 4)
