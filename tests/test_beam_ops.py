"""beam_select and beam_reorder against plain 64-bit implementations: sizes from one beam and one continuation up, odd lengths, masks that
leave nothing, dead and finished beams, infinities and NaN, strides, gradients, captured graphs; their refusals (no GPU needed)."""
import ctypes
import itertools

import pytest
import torch

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
NEG = float("-inf")


# ---- the definitions, in 64 bits on the host ----------------------------------------------------------------------------------------
def select_ref(logits, scores, k, mask=None, finished=None, end=None, normalize=True):
    """[b, j, v], [b, j] -> scores, parents, tokens [b, k] and the table of all continuations"""
    x = logits.detach().double().cpu()
    b, j, v = x.shape
    s = torch.zeros(b, j, dtype=torch.float64) if scores is None else scores.detach().double().cpu()
    keep = torch.ones(b, j, v, dtype=torch.bool) if mask is None else mask.cpu().expand(b, j, v)
    x = x.masked_fill(~keep, NEG)
    if normalize:
        x = x - torch.logsumexp(x, -1, keepdim=True)
    if finished is not None:
        only = torch.full((v,), NEG, dtype=torch.float64)
        only[end] = 0.0
        x = torch.where(finished.cpu()[..., None], only, x)
    c = s[..., None] + x
    c = torch.where(c.isnan(), NEG, c).view(b, j * v)
    order = torch.sort(c, dim=-1, descending=True, stable=True).indices[:, :k]
    return c.gather(1, order), order // v, order % v, c.view(b, j, v)


def check_select(step, ref):
    """Scores: a sum of at most |c| is rounded once to fp32 (half a step, 2^-24 |c|); the log-sum may carry 2^-20: its terms come from a
    32-bit exp (2 steps), a rounded argument (2 steps) and sums of at most 12 terms in 32 bits."""
    want, parents, tokens, _ = ref
    got = step.scores.detach().double().cpu()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin) and torch.equal(got[~fin], want[~fin])
    assert ((got - want)[fin].abs() <= want[fin].abs() * 2.0 ** -24 + 2.0 ** -20).all()
    assert torch.equal(step.parents.cpu(), parents) and torch.equal(step.tokens.cpu(), tokens)


def make(b, j, v, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    lg = (torch.randn(b, j, v, generator=g) * spread).to(DT[dtype]).cuda()
    return lg, (-torch.rand(b, j, generator=g).cumsum(-1) * 0.3).cuda()


SIZES = [(1, 1, 1, 1), (3, 1, 7, 7), (5, 4, 4, 4), (2, 3, 1, 2), (2, 8, 8, 64), (1, 64, 3, 5), (4, 7, 33, 13), (3, 5, 257, 5), (2, 2, 1024, 64),
         (2, 6, 1023, 6), (1, 3, 2049, 8), (2, 3, 5001, 16), (1, 2, 32003, 33), (1, 1, 100001, 4), (1, 4, 131072, 8), (67, 4, 4, 4), (300, 2, 65, 3),
         (1030, 1, 130, 2), (2, 64, 64, 64), (9, 16, 16, 16), (5, 13, 19, 13), (300, 1, 65, 64), (3, 9, 57, 20), (7, 32, 32, 32), (2, 33, 47, 40), (2, 64, 32, 64),
         (3, 4, 1024, 64), (2, 5, 819, 7), (2, 64, 65, 64), (1, 64, 700, 64), (1, 40, 5000, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("b,j,v,k", SIZES)
def test_select(dev, b, j, v, k, normalize, dtype):
    import vector_quantize_pytorch_amd as A
    lg, sc = make(b, j, v, dtype, seed=v)
    check_select(A.beam_select(lg, sc, k, normalize=normalize), select_ref(lg, sc, k, normalize=normalize))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("b,j,v,k", [(4, 4, 5, 7), (3, 5, 40, 9), (3, 9, 90, 12), (3, 8, 500, 33), (2, 6, 1000, 6), (2, 3, 9000, 64), (1, 4, 70001, 5), (70, 8, 9000, 8)])
@pytest.mark.parametrize("kind", ["lowest", "infinite", "one", "first", "finished", "masked"])
def test_select_scores_that_hide_logits(dev, b, j, v, k, kind, dtype):
    """scores beside which 64 bits do not see the logits: all continuations of such a beam are equal, and their places decide.  one: only
    the last beam has such a score; first: the first beam has an ordinary one; finished: it has ended, one continuation is left to it"""
    import vector_quantize_pytorch_amd as A
    lg, sc = make(b, j, v, dtype, seed=3)
    low = torch.finfo(torch.float32).min
    finished = mask = None
    if kind == "one":
        sc[:, -1] = 1e30
    else:
        sc[:, 0 if kind in ("lowest", "infinite", "masked") else 1:] = float("inf") if kind == "infinite" else low
    if kind == "finished":
        finished = torch.zeros(b, j, dtype=torch.bool, device="cuda")
        finished[:, 0] = True
        finished[0, -1] = True
    if kind == "masked":
        mask = torch.rand(b, j, v, generator=torch.Generator().manual_seed(4)).cuda() < 0.1
    for normalize in (True, False):
        step = A.beam_select(lg, sc, k, mask=mask, finished=finished, end_token=None if finished is None else v // 2, normalize=normalize)
        check_select(step, select_ref(lg, sc, k, mask=mask, finished=finished, end=v // 2, normalize=normalize))


@pytest.mark.gpu
@pytest.mark.parametrize("v,k", [(300, 5), (2500, 40), (40000, 8)])
def test_select_logits_that_scores_hide(dev, v, k):
    """logits around 0 that differ by 2^-80: beside a score of -1 they are equal, beside a score of 0 they are not"""
    import vector_quantize_pytorch_amd as A
    g = torch.Generator().manual_seed(v)
    lg = (torch.randn(2, 3, v, generator=g) * 2.0 ** -80).cuda()
    lg[0, 2, v - 3] = 1.0
    for sc in (torch.full((2, 3), -1.0), torch.tensor([[0.0, -1.0, -1.0], [-1.0, 0.0, 0.0]]), torch.tensor([[0.0, -1.0, -2.0], [-1.0, 2.0 ** -81, 0.0]])):
        check_select(A.beam_select(lg, sc.cuda(), k, normalize=False), select_ref(lg, sc, k, normalize=False))


@pytest.mark.gpu
@pytest.mark.parametrize("b,j,v,k", [(3, 4, 4, 5), (2, 5, 1000, 6), (2, 3, 40009, 9), (3, 5, 50, 6), (4, 5, 100, 6), (2, 7, 250, 20), (2, 5, 800, 9)])
@pytest.mark.parametrize("kind", ["row", "shared", "each", "beam", "nothing"])
def test_select_masked(dev, b, j, v, k, kind):
    """what the mask leaves out holds NaN and infinities; `nothing`: one beam, and one whole entry, have no continuation"""
    import vector_quantize_pytorch_amd as A
    lg, sc = make(b, j, v, "bf16", seed=5)
    g = torch.Generator().manual_seed(6)
    shape = dict(row=(v,), shared=(1, 1, v), each=(b, j, v), beam=(b, j, 1), nothing=(b, j, v))[kind]
    mask = torch.rand(shape, generator=g) < 0.6
    if kind == "nothing":
        mask[0, 1:3] = False
        mask[1] = False
    full = mask.expand(b, j, v)
    junk = torch.tensor([float("nan"), float("inf"), NEG])[torch.randint(0, 3, (b, j, v), generator=g)]
    lg = torch.where(full.cuda(), lg, junk.cuda().to(lg.dtype))
    mask = mask.cuda()
    for norm in (True, False):
        ref = select_ref(lg.masked_fill(~mask, 0.0), sc, k, mask=mask, normalize=norm)
        check_select(A.beam_select(lg, sc, k, mask=mask, normalize=norm), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [5, 40, 300, 700, 33333])
def test_select_dead_finished_and_not_a_number(dev, v):
    import vector_quantize_pytorch_amd as A
    b, j, k, end = 4, 6, 9, v // 2
    lg, sc = make(b, j, v, "fp32", seed=v)
    sc[0, 1:] = NEG                                        # one live beam
    sc[1, 2] = float("nan")
    lg[1, 0, v // 3] = float("nan")
    lg[1, 1, v - 1] = float("inf")
    lg[1, 3] = NEG
    lg[2, 0, :] = torch.finfo(torch.float32).min           # the type's lowest value is a number
    lg[2, 1, 1:] = NEG
    fin = torch.zeros(b, j, dtype=torch.bool, device="cuda")
    fin[3, :4] = True
    fin[1, 5] = True
    lg[3, 1] = float("nan")                                # a finished beam's logits are not used
    for norm in (True, False):
        f = fin.clone()
        ref_lg = torch.where(lg.isnan() & f[..., None], 0.0, lg)
        check_select(A.beam_select(lg, sc, k, finished=f, end_token=end, normalize=norm),
                     select_ref(ref_lg, sc, k, finished=f, end=end, normalize=norm))
    none = A.beam_select(torch.full((2, 3, v), NEG, device="cuda"), None, 4)
    assert (none.scores == NEG).all() and torch.equal(none.parents * v + none.tokens, torch.arange(4, device="cuda").expand(2, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("j,v,k", [(3, 5, 15), (4, 1500, 64), (2, 50000, 64), (5, 9001, 7), (16, 16, 16), (4, 100, 7), (8, 120, 64), (7, 250, 64), (5, 800, 64), (64, 64, 3)])
def test_select_ties(dev, j, v, k):
    """equal continuations survive by ascending place: a constant table, few values, runs in ascending and descending order"""
    import vector_quantize_pytorch_amd as A
    n = torch.arange(v, device="cuda").float()
    g = torch.Generator(device="cuda").manual_seed(1)
    few = torch.randint(0, 3, (j, v), generator=g, device="cuda").float()
    table = torch.stack([torch.zeros(j, v, device="cuda"), few, (n / 64).floor().expand(j, v), (-n / 64).floor().expand(j, v)])
    check_select(A.beam_select(table, None, k, normalize=False), select_ref(table, None, k, normalize=False))
    alike = table[:1].bfloat16()
    check_select(A.beam_select(alike, None, k), select_ref(alike, None, k))
    same = torch.randn(1, 1, v, generator=g, device="cuda").expand(1, j, v)            # all beams alike (stride 0)
    check_select(A.beam_select(same, None, k), select_ref(same, None, k))


@pytest.mark.gpu
def test_select_layouts(dev):
    """leading dims, rows inside a wider tensor, a transposed table, odd starts, a scalar lead"""
    import vector_quantize_pytorch_amd as A
    wide = torch.randn(3, 2, 4, 999, device="cuda").bfloat16()
    for lg in (wide, wide[..., 1:700], wide[:, :, 1:3], wide[:, 1], wide.transpose(0, 2), wide[0, 0], wide[..., ::3]):
        j, v = lg.shape[-2:]
        sc = -torch.rand(lg.shape[:-1], device="cuda")
        step = A.beam_select(lg, sc, 5)
        ref = select_ref(lg.reshape(-1, j, v), sc.reshape(-1, j), 5)
        assert step.scores.shape == (*lg.shape[:-2], 5)
        check_select(A.BeamStep(*(t.reshape(-1, 5) for t in step)), ref)
    empty = A.beam_select(torch.empty(0, 3, 10, device="cuda"), torch.empty(0, 3, device="cuda"), 2)
    assert empty.scores.shape == (0, 2) and empty.tokens.dtype == torch.int64


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("b,j,v,k", [(1, 1, 1, 1), (3, 4, 4, 6), (2, 5, 257, 9), (2, 3, 9001, 16), (1, 2, 40003, 64), (70, 16, 16, 16), (3, 64, 64, 64), (3, 7, 130, 33)])
def test_select_gradient(dev, b, j, v, k, normalize, dtype):
    """Against the formula in 64 bits.  The softmax carries 2^-19 of itself (the log-sum's 2^-20 and a 32-bit exp), the sum over the
    kept ones k steps of 2^-24, the result is rounded once to its type."""
    import vector_quantize_pytorch_amd as A
    lg, sc = make(b, j, v, dtype, seed=v + 1)
    g = torch.Generator().manual_seed(3)
    mask = (torch.rand(b, j, v, generator=g) < 0.9).cuda()
    mask[..., 0] = True
    fin = (torch.rand(b, j, generator=g) < 0.2).cuda()
    sc[0, -1] = NEG
    w = torch.randn(b, k, generator=g).cuda()
    lg.requires_grad_(True)
    sc.requires_grad_(True)
    step = A.beam_select(lg, sc, k, mask=mask, finished=fin, end_token=v - 1, normalize=normalize)
    dl, ds = torch.autograd.grad(step.scores, (lg, sc), w)
    vals, par, tok, _ = select_ref(lg, sc, k, mask=mask, finished=fin, end=v - 1, normalize=normalize)
    gw = torch.where(vals > NEG, w.cpu().double(), 0.0)
    want_s, size_s = torch.zeros(b, j, dtype=torch.float64), torch.zeros(b, j, dtype=torch.float64)
    want_s.scatter_add_(1, par, gw)
    size_s.scatter_add_(1, par, gw.abs())
    want = torch.zeros(b, j * v, dtype=torch.float64).scatter_add_(1, par * v + tok, gw).view(b, j, v)
    p = torch.zeros(b, j, v, dtype=torch.float64)
    if normalize:
        p = lg.detach().cpu().double().masked_fill(~mask.cpu(), NEG).softmax(-1)
        want = want - p * want_s[..., None]
    want = want.masked_fill(fin.cpu()[..., None], 0.0)
    tol = torch.finfo(DT[dtype]).eps / 2 * want.abs() + size_s[..., None] * (p * 2.0 ** -19 + (want != 0) * k * 2.0 ** -24) + (2.0 ** -24 if dtype == "fp16" else 0)
    assert dl.dtype == DT[dtype] and dl.shape == lg.shape
    assert ((dl.cpu().double() - want).abs() <= tol).all()
    assert ((ds.cpu().double() - want_s).abs() <= size_s * k * 2.0 ** -24).all()


@pytest.mark.gpu
def test_select_gradient_against_differences(dev):
    """f(h) = sum w scores along a direction u with |u| <= 1: a central difference at h = 2^-5 is off by h^2/6 |f'''| <= 2^-10/6 * 2 * sum|w|
    (third cumulants of a softmax are at most 1, the accumulated score is linear) and by the 2^-20 + 2^-24 |c| of each score over 2 h"""
    import vector_quantize_pytorch_amd as A
    lg, sc = make(1, 3, 50, "fp32", seed=11, spread=1.0)
    for jj, t in itertools.product(range(3), range(2)):
        lg[0, jj, 7 * jj + t] = 6.0 + 0.9 * t
    sc = torch.tensor([[0.0, -3.0, -6.0]], device="cuda")
    w, h = torch.randn(1, 6, device="cuda"), 2.0 ** -5
    lg.requires_grad_(True)
    sc.requires_grad_(True)
    u = (torch.rand(1, 3, 50, device="cuda") * 2 - 1, torch.rand(1, 3, device="cuda") * 2 - 1)
    step = A.beam_select(lg, sc, 6)
    dl, ds = torch.autograd.grad(step.scores, (lg, sc), w)
    ends = []                                               # the scores of the six places on either side, in whatever order they survive there
    for s in (-1, 1):
        near = A.beam_select((lg + s * h * u[0]).detach(), (sc + s * h * u[1]).detach(), 60)
        place = (near.parents * 50 + near.tokens) == (step.parents * 50 + step.tokens)[0, :, None]
        assert (place.sum(-1) == 1).all()
        ends.append(near.scores[0, place.int().argmax(-1)].double())
    diff = ((ends[1] - ends[0]) * w[0]).sum().item() / (2 * h)
    have = ((dl.double() * u[0]).sum() + (ds.double() * u[1]).sum()).item()
    aw = w.abs().sum().item()
    assert abs(diff - have) <= aw * (2.0 ** -10 / 3 + 2 * (2.0 ** -20 + 2.0 ** -24 * 16) / (2 * h) + 2.0 ** -16)


@pytest.mark.gpu
@pytest.mark.parametrize("j,v", [(4, 4), (4, 3000), (3, 70001)])
def test_select_in_a_graph_and_on_another_stream(dev, j, v):
    """two captured graphs replayed in turn with eager work between, each replay like the eager result; a side stream"""
    import vector_quantize_pytorch_amd as A
    lgs = [make(3, j, v, "bf16", seed=s) for s in (1, 2)]
    A.beam_select(*lgs[0], 4)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for lg, sc in lgs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(A.beam_select(lg, sc, 4))
        graphs.append(g)
    for r in range(3):
        for i, (g, o) in enumerate(zip(graphs, outs)):
            lgs[i][0].copy_(make(3, j, v, "bf16", seed=10 * r + i)[0])
            g.replay()
            eager = A.beam_select(*lgs[i], 4)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(o, eager))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = A.beam_select(*lgs[0], 4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, A.beam_select(*lgs[0], 4)))


# ---- reordering ---------------------------------------------------------------------------------------------------------------------
def reorder_ref(s, par):
    """host gather, zeros for parents outside the beams"""
    lead, j = par.shape[:-1], s.shape[par.ndim - 1]
    flat = s.detach().cpu().flatten(0, par.ndim - 2) if par.ndim > 1 else s.detach().cpu()[None]
    p = par.cpu().reshape(-1, par.shape[-1])
    out = flat[torch.arange(len(p))[:, None], p.clamp(0, j - 1)]
    out[(p < 0) | (p >= j)] = 0
    return out.reshape(*lead, p.shape[-1], *s.shape[par.ndim:])


@pytest.mark.gpu
@pytest.mark.parametrize("b,j,k", [(1, 1, 1), (3, 4, 4), (2, 1, 8), (5, 8, 3), (33, 2, 2)])
def test_reorder(dev, b, j, k):
    """many types and row sizes in one call, parents repeated, left out, and outside the beams"""
    import vector_quantize_pytorch_amd as A
    g = torch.Generator().manual_seed(b)
    par = torch.randint(-1, j + 1, (b, k), generator=g).cuda()
    shapes = [(), (1,), (3,), (16,), (5, 7), (8, 33, 64), (2, 1000), (65,), (4099,)]
    types = [torch.float32, torch.bfloat16, torch.int64, torch.uint8, torch.float64, torch.bool, torch.float16, torch.complex64]
    states = [torch.randint(0, 100, (b, j, *s), generator=g).to(t).cuda() for s, t in itertools.product(shapes, types)]
    new = A.beam_reorder(states, par)
    for s, n in zip(states, new):
        assert n.dtype == s.dtype and torch.equal(n.cpu(), reorder_ref(s, par))
    out = [torch.full_like(n, 7) for n in new]
    same = A.beam_reorder(states, par, out=out)
    assert all(a is o and torch.equal(a, n) for a, o, n in zip(same, out, new))


@pytest.mark.gpu
def test_reorder_layouts(dev):
    """leading dims, caches cut to a length, odd offsets, transposed and expanded states, empty ones"""
    import vector_quantize_pytorch_amd as A
    par = torch.randint(0, 4, (3, 2, 5), device="cuda")
    base = torch.randn(3, 2, 4, 6, 40, 9, device="cuda")
    half = base.bfloat16()
    states = [base, base[..., :17, :], half[..., 1:8], base.transpose(-1, -2), base[:, :, :, ::2], base[:, :, :, 0, 0, 0], half[:, :, :, 1:5, 3:30],
              torch.randn(2, 3, 4, 8, device="cuda").transpose(0, 1), torch.randn(4, 3, 2, 8, device="cuda").permute(1, 2, 0, 3),
              torch.randn(3, 2, 1, 8, device="cuda").expand(3, 2, 4, 8), torch.randn(3, 2, 4, 1, device="cuda").expand(3, 2, 4, 8), base[..., :0]]
    for s, n in zip(states, A.beam_reorder(states, par)):
        assert torch.equal(n.cpu(), reorder_ref(s, par))
    assert A.beam_reorder([], par) == []
    none = A.beam_reorder([torch.empty(0, 3, 5, device="cuda")], torch.empty(0, 2, dtype=torch.int64, device="cuda"))
    assert none[0].shape == (0, 2, 5)
    flat = torch.randn(4, 3, device="cuda")                                    # no leading dim
    assert torch.equal(A.beam_reorder([flat], torch.tensor([3, 3, 0], device="cuda"))[0], flat[[3, 3, 0]])


@pytest.mark.gpu
def test_reorder_beyond_32_bit_offsets(dev):
    """a cache of more than 2^32 bytes: the last rows come from, and go, behind that border"""
    import vector_quantize_pytorch_amd as A
    s = torch.zeros(3, 2, 400_000_001, dtype=torch.bfloat16, device="cuda")       # 4.8 GB
    for i in range(6):
        s[i // 2, i % 2, -1], s[i // 2, i % 2, 0] = i + 1, 10 + i
    par = torch.tensor([[1, 0], [0, 0], [1, 1]], device="cuda")
    n, = A.beam_reorder([s], par)
    assert n[..., -1].tolist() == [[2, 1], [3, 3], [6, 6]] and n[..., 0].tolist() == [[11, 10], [12, 12], [15, 15]]
    assert int((n != 0).sum()) == 12


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("b,j,k,shape", [(1, 1, 1, (1,)), (3, 4, 6, (7, 5)), (50, 4, 4, (256,)), (2, 8, 3, (3, 1025)), (2, 3, 64, (9,))])
def test_reorder_gradient(dev, b, j, k, shape, dtype):
    """the sum of at most k gradients in 32 bits (k - 1 half steps of 2^-24), rounded once; beams nobody continues get zeros"""
    import vector_quantize_pytorch_amd as A
    g = torch.Generator().manual_seed(k)
    par = torch.randint(-1, j, (b, k), generator=g).cuda()
    s = torch.randn(b, j, *shape, generator=g).to(DT[dtype]).cuda().requires_grad_(True)
    frozen = torch.arange(b * j).view(b, j).cuda()
    still = torch.randn(b, j, 3, generator=g).cuda()
    n, f, st = A.beam_reorder([s, frozen, still], par)
    assert n.requires_grad and not f.requires_grad and not st.requires_grad
    w = torch.randn(n.shape, generator=g).to(DT[dtype]).cuda()
    d, = torch.autograd.grad(n, s, w)
    want, size = torch.zeros(s.shape, dtype=torch.float64), torch.zeros(s.shape, dtype=torch.float64)
    for bb, i in itertools.product(range(b), range(k)):
        if par[bb, i] >= 0:
            want[bb, par[bb, i]] += w[bb, i].cpu().double()
            size[bb, par[bb, i]] += w[bb, i].cpu().double().abs()
    tol = torch.finfo(DT[dtype]).eps / 2 * want.abs() + size * k * 2.0 ** -24 * (1 + torch.finfo(DT[dtype]).eps) + (2.0 ** -25 if dtype == "fp16" else 0)
    assert d.dtype == s.dtype and ((d.cpu().double() - want).abs() <= tol).all()


@pytest.mark.gpu
def test_reorder_many_states_in_a_graph(dev):
    import vector_quantize_pytorch_amd as A
    states = [torch.randn(2, 3, 5 + i, device="cuda") for i in range(71)]          # more than one launch takes
    par = torch.randint(0, 3, (2, 4), device="cuda")
    out = [torch.empty(2, 4, 5 + i, device="cuda") for i in range(71)]
    A.beam_reorder(states, par, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        A.beam_reorder(states, par, out=out)
    for r in range(3):
        par.copy_(torch.randint(0, 3, (2, 4), generator=torch.Generator().manual_seed(r)))
        for o in out:
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o.cpu(), reorder_ref(s, par)) for s, o in zip(states, out))


# ---- the residual quantizer's beam search on these operators ---------------------------------------------------------------------------
def plain_beam_search(rvq, x, beam, mask=None, drop_at=None):
    """every continuation formed, then the kept ones picked; equal totals by place (stable sort)"""
    lead, last = x.shape[:-1], len(rvq.layers) - 1 if drop_at is None else drop_at
    scores = torch.zeros(*lead, 1, device=x.device)
    residual, out = x[..., None, :], torch.zeros_like(x)[..., None, :]
    idxs, losses = torch.empty(*lead, 1, 0, dtype=torch.long, device=x.device), torch.empty(*lead, 1, 0, device=x.device)
    for qi, vq in enumerate(rvq.layers):
        if qi > last:
            idxs, losses = torch.nn.functional.pad(idxs, (0, 1), value=-1), torch.nn.functional.pad(losses, (0, 1))
            continue
        q, ind, loss = vq(residual, mask=mask, topk=beam)
        k = ind.shape[-1]
        scores = (scores[..., None] - loss.detach() * rvq.beam_score_weights[qi]).flatten(-2)
        step = q.detach() if rvq.quant_grad_frac <= 0 else rvq.quant_grad_frac * q + (1 - rvq.quant_grad_frac) * q.detach()
        residual = (residual[..., None, :] - step).flatten(-3, -2)
        out = (out[..., None, :] + q).flatten(-3, -2)
        idxs = torch.cat((idxs[..., None, :].expand(*idxs.shape[:-1], k, -1), ind[..., None]), -1).flatten(-3, -2)
        losses = torch.cat((losses[..., None, :].expand(*losses.shape[:-1], k, -1), loss[..., None].float()), -1).flatten(-3, -2)
        keep = beam if qi != last else 1
        if scores.shape[-1] > keep:
            scores, order = scores.sort(dim=-1, descending=True, stable=True)
            scores, order = scores[..., :keep], order[..., :keep]
            residual, out = (t.gather(-2, order[..., None].expand(*order.shape, t.shape[-1])) for t in (residual, out))
            idxs, losses = (t.gather(-2, order[..., None].expand(*order.shape, t.shape[-1])) for t in (idxs, losses))
    out, idxs, losses = out[..., 0, :], idxs[..., 0, :], losses[..., 0, :]
    if mask is not None:
        losses = torch.where(mask[..., None], losses, 0.0).flatten(0, -2).sum(0) / mask.sum().clamp_min(1e-4)
    else:
        losses = losses.flatten(0, -2).mean(0)
    return out, idxs, losses


@pytest.mark.gpu
@pytest.mark.parametrize("kw,beam", [(dict(), 2), (dict(quant_grad_frac=0.25), 4), (dict(masked=True), 3), (dict(shared_codebook=True, threshold_ema_dead_code=2), 3),
                                     (dict(quantize_dropout=True), 4), (dict(beam_score_quantizer_weights=[1.0, 0.5, 0.25, 2.0]), 5), (dict(bf16=True), 4), (dict(), 70)])
def test_residual_beam_search_matches_plain(dev, kw, beam):
    """the same values bit for bit; gradients add a beam's continuations in another order: 2^-20 of their size"""
    import copy

    import vector_quantize_pytorch_amd as A
    torch.manual_seed(beam)
    kw = dict(kw)
    masked, half = kw.pop("masked", False), kw.pop("bf16", False)
    a = A.ResidualVQ(dim=32, num_quantizers=4, codebook_size=96, beam_size=beam, **kw).cuda().train()
    b = copy.deepcopy(a)
    x = torch.randn(1, 90, 32, device="cuda").to(torch.bfloat16 if half else torch.float32)
    mask = (torch.arange(90, device="cuda") < 61)[None] if masked else None
    drop = None
    fw = dict(mask=mask)
    if kw.get("quantize_dropout"):
        import random
        fw["rand_quantize_dropout_fixed_seed"] = 5
        drop = random.Random(5).randrange(0, 4)
    xa, xb = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    got, want = a(xa, **fw), plain_beam_search(b, xb, beam, mask, drop)
    assert got[0].shape == x.shape and got[1].shape == (1, 90, 4) and got[2].shape == (4,)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0], want[0]) and torch.allclose(got[2], want[2], rtol=2.0 ** -20, atol=0.0)
    w = torch.randn(x.shape, device="cuda").to(x.dtype)
    ga, = torch.autograd.grad((got[0] * w).float().sum() + got[2].sum(), xa)
    gb, = torch.autograd.grad((want[0] * w).float().sum() + want[2].sum(), xb)
    assert (ga - gb).abs().max().item() <= (2.0 ** -5 if half else 2.0 ** -18) * gb.abs().max().item()


@pytest.mark.gpu
def test_residual_beam_search_needs_losses(dev):
    import vector_quantize_pytorch_amd as A
    r = A.ResidualVQ(dim=32, num_quantizers=2, codebook_size=32, beam_size=2).cuda()
    with pytest.raises(RuntimeError, match="commitment loss"):
        r.eval()(torch.randn(1, 8, 32, device="cuda"))


@pytest.mark.gpu
def test_reorder_of_conjugated_and_negated_states(dev):
    """torch's conj() and imag of it leave memory as it is and set a flag: the results are the tensors' values"""
    import vector_quantize_pytorch_amd as A
    z = torch.randn(3, 4, 6, 5, dtype=torch.complex64, device="cuda")
    par = torch.tensor([[1, 1, 3], [0, 2, -1], [3, 0, 0]], device="cuda")
    states = [z.conj(), z.conj().imag, z.conj()[..., 1:4], z.transpose(2, 3).conj(), torch._neg_view(z.real.contiguous()), z, z.mH]
    for s, n in zip(states, A.beam_reorder(states, par)):
        assert torch.equal(n.cpu(), reorder_ref(s.resolve_conj().resolve_neg(), par))
    out = [torch.empty(3, 3, *s.shape[2:], dtype=s.dtype, device="cuda") for s in states]
    A.beam_reorder(states, par, out=out)
    for s, o in zip(states, out):
        assert torch.equal(o.cpu(), reorder_ref(s.resolve_conj().resolve_neg(), par))
    im = torch.randn(3, 4, 7, device="cuda", requires_grad=True)
    new, = A.beam_reorder([torch.complex(im, im).conj().imag], par)
    w = torch.randn(3, 3, 7, device="cuda")
    assert torch.equal(new.detach().cpu(), reorder_ref(-im, par))
    got, = torch.autograd.grad(new, im, torch._neg_view(w), retain_graph=True)
    back, = torch.autograd.grad(new, im, w)
    assert torch.equal(got, -back) and back.abs().sum() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("v", [1, 6, 300, 9000])
def test_select_of_negated_tensors(dev, v):
    import vector_quantize_pytorch_amd as A
    lg, sc = make(3, 4, v, "fp32", seed=v)
    k = min(5, 4 * v)
    ref = select_ref(lg, sc, k)
    for a, b in ((torch._neg_view(-lg), sc), (lg, torch._neg_view(-sc)), (torch.complex(lg, -lg).conj().imag, torch.complex(sc, -sc).conj().imag)):
        check_select(A.beam_select(a, b, k), ref)
    lg.requires_grad_(True)
    w = torch.randn(3, k, device="cuda")
    step = A.beam_select(lg, sc, k)
    got, = torch.autograd.grad(step.scores, lg, torch._neg_view(-w), retain_graph=True)
    assert torch.equal(got, torch.autograd.grad(step.scores, lg, w)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("lead,j,v", [((3,), 4, 4), ((3,), 4, 3000), ((2, 2), 5, 50)])
def test_tokens_may_be_edited_between_selection_and_backward(dev, lead, j, v):
    """parents, tokens and scores are tensors of their own: the backward of a reordering needs the parents alone"""
    import vector_quantize_pytorch_amd as A
    lg = torch.randn(*lead, j, v, device="cuda")
    state = torch.randn(*lead, j, 6, device="cuda", requires_grad=True)
    step = A.beam_select(lg, None, 4)
    assert len({t.data_ptr() for t in step}) == 3 and all(t.is_contiguous() for t in step)
    new, = A.beam_reorder([state], step.parents)
    parents = step.parents.clone()
    step.tokens.masked_fill_(step.tokens == v - 1, 0)
    step.scores.zero_()
    new.sum().backward()
    want = torch.zeros(*lead, j, device="cuda").scatter_add_(-1, parents, torch.ones(*lead, 4, device="cuda"))
    assert torch.equal(state.grad, want[..., None].expand_as(state))


@pytest.mark.gpu
@pytest.mark.parametrize("b,j,v,k", [(2 ** 23 + 5, 2, 2, 3), (2 ** 23 + 5, 1, 65, 2), (2 ** 23 + 5, 3, 30, 4), (2 ** 18 + 1, 64, 64, 64), (2 ** 17 + 1, 64, 65, 3), (2 ** 20 + 1, 8, 513, 5)])
def test_select_of_large_batches(dev, b, j, v, k):
    """batches that take several launches, or more entries than a launch has tiles: the entries on either side of every border, forward and
    backward, against the same entries alone (their tiles differ, so the log-sums' last bits may)"""
    import vector_quantize_pytorch_amd as A
    g = torch.Generator(device="cuda").manual_seed(j)
    lg = torch.empty(b, j, v, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    sc = torch.randn(b, j, generator=g, device="cuda")
    mask = torch.rand(b, 1, v, generator=g, device="cuda") < 0.8
    fin = torch.rand(b, j, generator=g, device="cuda") < 0.1
    some = sorted({n for per in (1, j, 2 * j) for m in (1, 2) for n in (0, 1, 2 ** 23 // per * m - 1, 2 ** 23 // per * m, b - 1) if n < b})
    some = torch.tensor(some, device="cuda")
    lg.requires_grad_(True)
    sc.requires_grad_(True)
    step = A.beam_select(lg, sc, k, mask=mask, finished=fin, end_token=v - 1)
    w = torch.randn(b, k, generator=g, device="cuda")
    dl, ds = torch.autograd.grad(step.scores, (lg, sc), w)
    l1, s1 = lg.detach()[some].requires_grad_(True), sc.detach()[some].requires_grad_(True)
    alone = A.beam_select(l1, s1, k, mask=mask[some], finished=fin[some], end_token=v - 1)
    d1, e1 = torch.autograd.grad(alone.scores, (l1, s1), w[some])
    check_select(alone, select_ref(l1, s1, k, mask=mask[some], finished=fin[some], end=v - 1))
    assert torch.equal(step.parents[some], alone.parents) and torch.equal(step.tokens[some], alone.tokens) and torch.equal(ds[some], e1)
    real = alone.scores > NEG
    assert torch.equal(step.scores[some] > NEG, real) and ((step.scores[some] - alone.scores)[real].abs() <= 2.0 ** -20 * (1 + alone.scores[real].abs())).all()
    assert ((dl[some].float() - d1.float()).abs() <= 2.0 ** -7 * d1.float().abs()).all()       # (one step of bf16)
    assert not ((step.parents < 0) | (step.parents >= j) | (step.tokens < 0) | (step.tokens >= v)).any()


@pytest.mark.gpu
def test_reorder_of_more_than_2_31_rows(dev):
    """the continuations of a residual beam search: 2^19 entries of 64 x 64; parents that differ, so that every gradient lies alone"""
    import vector_quantize_pytorch_amd as A
    b, j = 2 ** 19 + 3, 4096
    g = torch.Generator(device="cuda").manual_seed(0)
    s = torch.empty(b, j, dtype=torch.bfloat16, device="cuda").normal_(generator=g).requires_grad_(True)
    par = torch.randint(0, j // 2, (b, 2), generator=g, device="cuda")
    par[:, 1] += j // 2
    par[-1] = torch.tensor([j - 1, 0])
    n, = A.beam_reorder([s], par)
    assert torch.equal(n, s.detach().gather(1, par))
    w = torch.rand(b, 2, generator=g, device="cuda").bfloat16() + 1
    d, = torch.autograd.grad(n, s, w)
    assert torch.equal(d.gather(1, par), w) and int(torch.count_nonzero(d)) == 2 * b


@pytest.mark.gpu
@pytest.mark.parametrize("j,v", [(4, 5), (4, 300), (4, 3000), (5, 20011)])
def test_select_log_sums(dev, j, v):
    """the C entry's log-sums: the admitted logits' own, NaN for beams whose logits are not used (finished, or without a score), not finite where
    nothing is left -- also in memory that held numbers before"""
    from vector_quantize_pytorch_amd.beam import _select
    lg, sc = make(3, j, v, "fp32", seed=v)
    mask = torch.rand(3, j, v, generator=torch.Generator().manual_seed(1)).cuda() < 0.7
    mask[..., 0] = True
    mask[2, 1] = False
    fin = torch.zeros(3, j, dtype=torch.bool, device="cuda")
    fin[0, 1] = fin[1, 0] = True
    sc[0, 2], sc[1, 3] = NEG, float("nan")
    for _ in range(2):
        held = [torch.full((n,), 1.0, dtype=torch.float64, device="cuda") for n in (3 * j, 64, 3 * j * 70)]
        del held
        *_, lse = _select(lg, sc, mask.view(torch.uint8), fin.view(torch.uint8), 4, v - 1, True, True)
        dead = fin | ~(sc > NEG)
        assert lse.shape == (3, j) and lse[dead].isnan().all()
        want = lg.double().masked_fill(~mask, NEG).logsumexp(-1)
        none = ~mask.any(-1)
        assert not torch.isfinite(lse[none]).any()
        assert ((lse - want)[~dead & ~none].abs() <= 2.0 ** -20).all()


@pytest.mark.gpu
def test_forward_mode_through_the_backward_is_refused(dev):
    """a gradient with a tangent (forward over backward): the backward's result would come without one"""
    import torch.autograd.forward_ad as fwad
    import vector_quantize_pytorch_amd as A
    from vector_quantize_pytorch_amd._lib import VQHipError
    lg, x = torch.randn(2, 3, 10, device="cuda", requires_grad=True), torch.randn(2, 3, 8, device="cuda", requires_grad=True)
    for y, t in ((A.beam_select(lg, None, 4).scores, lg), (A.beam_reorder([x], torch.zeros(2, 4, dtype=torch.int64, device="cuda"))[0], x), (A.group_norm(x, 2), x)):
        with fwad.dual_level():
            g = fwad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(VQHipError, match="forward-mode"):
                torch.autograd.grad(y, t, g, retain_graph=True)
        assert torch.autograd.grad(y, t, torch.ones_like(y))[0].shape == t.shape


# ---- refusals (host side: no GPU) ---------------------------------------------------------------------------------------------------
def test_select_refusals():
    import vector_quantize_pytorch_amd as A
    from vector_quantize_pytorch_amd._lib import VQHipError
    lg, sc = torch.zeros(2, 3, 10), torch.zeros(2, 3)
    for match, call in [
            ("no CPU fallback", lambda: A.beam_select(lg, sc, 4)),
            ("unsupported dtype", lambda: A.beam_select(lg.double(), sc, 4)),
            ("unsupported dtype", lambda: A.beam_select(lg.long(), sc, 4)),
            ("expected", lambda: A.beam_select(lg[0, 0], None, 4)),
            ("scores", lambda: A.beam_select(lg, sc[:, :2], 4)),
            ("scores", lambda: A.beam_select(lg, sc.bfloat16(), 4)),
            ("mask of", lambda: A.beam_select(lg, sc, 4, mask=torch.ones(10))),
            ("broadcast", lambda: A.beam_select(lg, sc, 4, mask=torch.ones(9, dtype=torch.bool))),
            ("finished", lambda: A.beam_select(lg, sc, 4, finished=torch.zeros(2, 3), end_token=1)),
            ("end_token", lambda: A.beam_select(lg, sc, 4, finished=torch.zeros(2, 3, dtype=torch.bool))),
            ("end_token", lambda: A.beam_select(lg, sc, 4, finished=torch.zeros(2, 3, dtype=torch.bool), end_token=10)),
            ("survivors", lambda: A.beam_select(lg, sc, 0)),
            ("survivors", lambda: A.beam_select(lg, sc, 31)),
            ("survivors", lambda: A.beam_select(torch.zeros(1, 1, 1000), None, 65)),
            ("survivors", lambda: A.beam_select(torch.zeros(1, 65, 10), None, 4)),
            ("survivors", lambda: A.beam_select(torch.zeros(1, 2, 0), None, 1))]:
        with pytest.raises(VQHipError, match=match):
            call()


def test_reorder_refusals():
    import vector_quantize_pytorch_amd as A
    from vector_quantize_pytorch_amd._lib import VQHipError
    s, par = torch.zeros(2, 3, 8), torch.zeros(2, 4, dtype=torch.int64)
    out = torch.zeros(2, 4, 8)
    big = torch.zeros(2, 7, 8)
    for match, call in [
            ("no CPU fallback", lambda: A.beam_reorder([s], par)),
            ("no CPU fallback", lambda: A.beam_reorder([s], par, out=[out])),
            ("parents", lambda: A.beam_reorder([s], par.int())),
            ("parents", lambda: A.beam_reorder([s], par[:, :0])),
            ("state", lambda: A.beam_reorder([s, torch.zeros(2)], par)),
            ("state", lambda: A.beam_reorder([s, torch.zeros(3, 3, 8)], par)),
            ("state", lambda: A.beam_reorder([s, torch.zeros(2, 4, 8)], par)),
            ("state", lambda: A.beam_reorder([torch.zeros(2, 0, 8)], par)),
            ("unsupported dtype", lambda: A.beam_reorder([s.double().requires_grad_()], par)),
            ("require a gradient", lambda: A.beam_reorder([s.clone().requires_grad_()], par, out=[out])),
            ("results", lambda: A.beam_reorder([s], par, out=[out, out])),
            ("out", lambda: A.beam_reorder([s], par, out=[out.half()])),
            ("out", lambda: A.beam_reorder([s], par, out=[torch.zeros(2, 4, 9)])),
            ("out", lambda: A.beam_reorder([s], par, out=[torch.zeros(2, 8, 4).transpose(1, 2)])),
            ("shares memory", lambda: A.beam_reorder([big[:1, :3], s[:1]], par[:1], out=[big[:1, 2:6], out[:1]])),
            ("shares memory", lambda: A.beam_reorder([s, s], par, out=[out, out]))]:
        with pytest.raises(VQHipError, match=match):
            call()


def test_c_entry_refusals():
    from vector_quantize_pytorch_amd import _lib
    from vector_quantize_pytorch_amd.beam import _Select, _State
    L = _lib.lib()
    ok = dict(logits=8, dtype=0, B=1, J=2, V=5, stride_b=10, stride_j=5, normalize=1, K=3, out_scores=8, parents=8, tokens=8)
    for rc, change in [(-1, dict(dtype=3)), (-1, dict(dtype=-1)), (-1, dict(B=-1)), (-1, dict(J=0)), (-1, dict(V=0)), (-1, dict(K=0)), (-2, dict(K=11)),
                       (-2, dict(J=65)), (-2, dict(J=64, V=2 ** 26)), (-2, dict(V=2 ** 40)), (-2, dict(B=2 ** 31)), (-1, dict(logits=0)), (-1, dict(tokens=0)),
                       (-1, dict(finished=8, end_token=5)), (-1, dict(finished=8, end_token=-1)), (0, dict(B=0, logits=0))]:
        s = _Select(**{**ok, **change})
        assert L.vqhip_beam_select(ctypes.byref(s), None) == rc, change
    assert L.vqhip_beam_select(None, None) == -1
    big = dict(ok, V=5000, stride_j=5000)
    nws = L.vqhip_beam_select_workspace_bytes(1, 2, 5000, 3)
    for rc, ws, size in [(-1, None, 0), (-1, 16, nws - 1), (-3, 24, nws)]:
        s = _Select(**big, workspace=ws, workspace_bytes=size)
        assert L.vqhip_beam_select(ctypes.byref(s), None) == rc
    s = _Select(**ok)
    assert L.vqhip_beam_select_bwd(ctypes.byref(s), None, 8, 8, None) == -1              # no gradient
    assert L.vqhip_beam_select_bwd(ctypes.byref(s), 8, 8, 8, None) == -1                 # normalized, no log-sums
    st = (_State * 1)((8, 8, 32, 16, 1, 0, 16))
    for rc, args in [(-1, (st, 33, 8, 1, 2, 2)), (-1, (st, -1, 8, 1, 2, 2)), (-1, (st, 1, None, 1, 2, 2)), (-1, (None, 1, 8, 1, 2, 2)), (-1, (st, 1, 8, 1, 0, 2)),
                     (-1, (st, 1, 8, 1, 2, 0)), (-2, (st, 1, 8, 2 ** 31, 2, 2)), (0, (st, 0, None, 1, 2, 2)), (0, (st, 1, None, 0, 2, 2))]:
        assert L.vqhip_beam_reorder(*args, None) == rc, args
    bad = (_State * 1)((8, 8, 32, 16, -1, 0, 16))
    assert L.vqhip_beam_reorder(bad, 1, 8, 1, 2, 2, None) == -1
    nul = (_State * 1)((None, 8, 32, 16, 1, 0, 16))
    assert L.vqhip_beam_reorder(nul, 1, 8, 1, 2, 2, None) == -1
    dts = (ctypes.c_int64 * 1)(5)
    assert L.vqhip_beam_reorder_bwd(st, dts, 1, 8, 1, 2, 2, None) == -1
    assert L.vqhip_beam_reorder_bwd(st, None, 1, 8, 1, 2, 2, None) == -1
    odd = (_State * 1)((8, 8, 32, 16, 1, 0, 15))
    assert L.vqhip_beam_reorder_bwd(odd, (ctypes.c_int64 * 1)(1), 1, 8, 1, 2, 2, None) == -1


def test_reorder_refuses_flagged_results():
    """a result with a pending conjugation or negation would hold something else than what is written into its memory"""
    import vector_quantize_pytorch_amd as A
    from vector_quantize_pytorch_amd._lib import VQHipError
    z, par = torch.zeros(2, 3, 8, dtype=torch.complex64), torch.zeros(2, 4, dtype=torch.int64)
    for s, o in ((z, torch.zeros(2, 4, 8, dtype=torch.complex64).conj()), (z.real, torch._neg_view(torch.zeros(2, 4, 8)))):
        with pytest.raises(VQHipError, match="pending"):
            A.beam_reorder([s], par, out=[o])


def test_forward_mode_is_refused():
    """a dual tensor's tangent would be lost: no entry point has a forward-mode derivative (host side: no GPU)"""
    import torch.autograd.forward_ad as fwad
    import vector_quantize_pytorch_amd as A
    from vector_quantize_pytorch_amd._lib import VQHipError
    lg, sc, st, par = torch.zeros(2, 3, 10), torch.zeros(2, 3), torch.zeros(2, 3, 8), torch.zeros(2, 4, dtype=torch.int64)
    with fwad.dual_level():
        def dual(t):
            return fwad.make_dual(t, torch.ones_like(t))
        for call in (lambda: A.beam_select(dual(lg), sc, 4), lambda: A.beam_select(lg, dual(sc), 4), lambda: A.beam_reorder([st, dual(st)], par),
                     lambda: A.beam_reorder([dual(st)], par, out=[torch.zeros(2, 4, 8)]), lambda: A.beam_reorder([st], par, out=[dual(torch.zeros(2, 4, 8))]),
                     lambda: A.beam_select(dual(lg.clone().requires_grad_()), sc, 4)):
            with pytest.raises(VQHipError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(VQHipError, match="forward-mode"):
                call()
        with pytest.raises(VQHipError, match="no CPU fallback"):             # a level without a tangent is no hindrance
            A.beam_select(lg, sc, 4)
    with pytest.raises(VQHipError, match="forward-mode"):
        torch.func.jvp(lambda t: A.beam_select(t, sc, 4).scores, (lg,), (lg,))


def test_c_entry_takes_large_batches():
    """what a launch cannot hold goes in several: the batch has no limit below 2^31.  Sizes are checked before the workspace, whose alignment
    (-3) is checked before anything is launched"""
    from vector_quantize_pytorch_amd import _lib
    from vector_quantize_pytorch_amd.beam import _Select
    L = _lib.lib()
    for b, j, v in [(2 ** 20, 16, 16), (2 ** 19, 32, 32), (2 ** 18, 64, 64), (2 ** 31 - 1, 1, 1), (2 ** 26, 8, 8), (2 ** 25, 1, 4096), (2 ** 18, 64, 65), (2 ** 25, 2, 5000)]:
        nws = L.vqhip_beam_select_workspace_bytes(b, j, v, 4)
        assert nws < 2 ** 34
        s = _Select(logits=8, dtype=1, B=b, J=j, V=v, stride_b=j * v, stride_j=v, normalize=0, K=min(4, j * v), out_scores=8, parents=8, tokens=8, workspace=24, workspace_bytes=nws)
        assert L.vqhip_beam_select(ctypes.byref(s), None) == -3, (b, j, v)


def test_reorder_takes_many_rows():
    """sizes are checked before the states' pointers: -1 here is the null pointer"""
    from vector_quantize_pytorch_amd import _lib
    from vector_quantize_pytorch_amd.beam import _State
    L = _lib.lib()
    nul = (_State * 1)((None, 8, 4096 * 4, 4, 1, 0, 4))
    dts = (ctypes.c_int64 * 1)(0)
    for b, j, k in [(2 ** 19, 4096, 64), (2 ** 20, 4096, 1), (2 ** 31 - 1, 64, 1)]:
        assert L.vqhip_beam_reorder(nul, 1, 8, b, j, k, None) == -1
        assert L.vqhip_beam_reorder_bwd(nul, dts, 1, 8, b, j, k, None) == -1
    assert L.vqhip_beam_reorder(nul, 1, 8, 2 ** 25, 1, 64, None) == -2


def test_reorder_refuses_results_that_require_a_gradient():
    """their history would stay as it was beside other values: s + s, say, would go on passing gradients to s"""
    import vector_quantize_pytorch_amd as A
    from vector_quantize_pytorch_amd._lib import VQHipError
    st, par = torch.zeros(2, 3, 8), torch.zeros(2, 4, dtype=torch.int64)
    leaf = torch.zeros(2, 4, 8, requires_grad=True)
    for o in (leaf, leaf + leaf):
        with pytest.raises(VQHipError, match="requires a gradient"):
            A.beam_reorder([st], par, out=[o])
        with torch.no_grad(), pytest.raises(VQHipError, match="no CPU fallback"):          # (as torch's own out= takes them there)
            A.beam_reorder([st], par, out=[o])
