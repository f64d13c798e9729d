"""Gradient norm and clipping (pr_grad_norm, pr_grad_clip, pr_adam_step_clipped; pogs_amd.optim) against the formulas
in float64.

Tolerances.  u = 2^-24 is half a float32 step.  Norms are summed in float64 and rounded once: u, and 2^-40 for the sums.
A scaled gradient carries the roundings of the norm, of norm + 1e-6, of the quotient and of the product: 4 u; in 16 bits
half a step of its type more.  The first moment after one step, m + 0.1 (g - m), has two roundings of its own and 0.1
rounded: |error| <= 8 u max(|m|, |g|); the second, with g twice: 16 u max(v, g^2)."""
import ctypes
import math
from array import array

import pytest
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _params(grads):
    out = []
    for g in grads:
        p = torch.zeros_like(g).requires_grad_(True)
        p.grad = g
        out.append(p)
    return out


def _norm64(grads, kind):
    flat = torch.cat([g.detach().cpu().double().reshape(-1) for g in grads]) if grads else torch.zeros(0, dtype=torch.float64)
    if kind == math.inf:
        return flat.abs().max().item()
    return flat.abs().sum().item() if kind == 1 else flat.square().sum().sqrt().item()


# ---- without a GPU ----------------------------------------------------------------------------------------------------
def _table(rows):
    words = array("q")
    for ptr, numel, dtype, s in rows:
        words.extend((ptr, numel, dtype | s << 32))
    return words, ctypes.c_void_p(words.buffer_info()[0])


def test_entry_points_validate_without_a_gpu():
    from pogs_amd import _lib

    lib = _lib.load()
    assert lib.pr_grad_norm_max_sets() >= 16
    one, at = _table([(1024, 100, 0, 0)])
    need = lib.pr_grad_norm_scratch_bytes(at, 1, 1)
    assert need >= 8
    big, big_at = _table([(1024, 1 << 40, 0, 0)])
    assert lib.pr_grad_norm_scratch_bytes(big_at, 1, 1) == 0        # more than an address space of gradients
    two, two_at = _table([(1024, 100, 0, 0), (1 << 20, 100, 2, 3)])
    assert lib.pr_grad_norm_scratch_bytes(two_at, 2, 4) == need + 8  # one partial a tensor at least
    scratch = ctypes.create_string_buffer(4096)
    sc = ctypes.c_void_p((ctypes.addressof(scratch) + 7) & ~7)
    odd = ctypes.c_void_p(sc.value + 1)
    m = (ctypes.c_double * 40)(*[1.0] * 40)
    bad = [([(1024, 100, 3, 0)], 1, 1), ([(1024, -1, 0, 0)], 1, 1), ([(0, 4, 0, 0)], 1, 1), ([(1025, 4, 0, 0)], 1, 1),
           ([(1025, 4, 2, 0)], 1, 1), ([(1024, 4, 0, 1)], 1, 1), ([(1024, 4, 0, 1), (4096, 4, 0, 0)], 2, 2),
           ([(1024, 4, 0, 0)], 1, 0), ([(1024, 4, 0, 0)], 1, 1000), ([(1024, 4, 0, 0)], -1, 1)]
    for rows, n, n_sets in bad:
        keep, p = _table(rows)
        assert lib.pr_grad_norm(p, n, n_sets, 2, sc, 4000, sc, None) == -1, rows
        assert lib.pr_grad_clip(p, n, n_sets, 2, m, sc, 4000, sc, None) == -1, rows
        assert lib.pr_grad_norm_scratch_bytes(p, n, n_sets) == 0
    assert lib.pr_grad_norm(None, 1, 1, 2, sc, 4000, sc, None) == -1
    for kind in (0, 4):
        assert lib.pr_grad_norm(at, 1, 1, kind, sc, 4000, sc, None) == -1
        assert lib.pr_grad_clip(at, 1, 1, kind, m, sc, 4000, sc, None) == -1
    for buffers in ((sc, 4000, None), (None, 4000, sc), (odd, 4000, sc)):
        assert lib.pr_grad_norm(at, 1, 1, 2, *buffers, None) == -1
        assert lib.pr_grad_clip(at, 1, 1, 2, m, *buffers, None) == -1
    assert lib.pr_grad_norm(at, 1, 1, 2, sc, need - 1, sc, None) == -3
    assert lib.pr_grad_clip(at, 1, 1, 2, m, sc, need - 1, sc, None) == -3
    assert lib.pr_grad_clip(at, 1, 1, 2, None, sc, 4000, sc, None) == -1
    for limit in (-1.0, math.nan):
        assert lib.pr_grad_clip(at, 1, 1, 2, (ctypes.c_double * 1)(limit), sc, 4000, sc, None) == -1
    for rows in ([(1024, 100, 0, 0), (1024, 100, 0, 0)], [(1024, 100, 0, 0), (1422, 9, 2, 0)],
                 [(5000, 1, 2, 0), (1024, 100, 0, 0), (1420, 1, 0, 0)]):
        keep, p = _table(rows)
        assert lib.pr_grad_clip(p, len(rows), 1, 2, m, sc, 4000, sc, None) == -2
        assert b"share memory" in lib.pr_last_hip_error()
    # the clipped step
    good = _lib.AdamGroup(1024, 1024, 1024, 1024, 8, 1, 1e-3, 0.9, 0.999, 1e-15)

    def step(group=good, rule=(0, 1.0), n=1, sets=1, scratch=sc, nbytes=4000, norms=sc):
        g, c = (_lib.AdamGroup * 1)(group), (_lib.ClipRule * 1)(_lib.ClipRule(rule[0], 0, rule[1]))
        return lib.pr_adam_step_clipped(g, c, n, sets, scratch, nbytes, norms, None)

    assert lib.pr_adam_step_clipped(None, None, 0, 1, None, 0, None, None) == 0
    assert lib.pr_adam_step_clipped(None, None, 1, 1, sc, 4000, sc, None) == -1
    for kw in (dict(n=-1), dict(rule=(0, -1.0)), dict(rule=(0, math.nan)), dict(rule=(1, 1.0)), dict(sets=0), dict(sets=1000),
               dict(scratch=None), dict(scratch=odd), dict(norms=None),
               dict(group=_lib.AdamGroup(1024, 1024, 1024, 1024, 8, 0, 1e-3, 0.9, 0.999, 1e-15)),
               dict(group=_lib.AdamGroup(1024, 1028, 1024, 1024, 8, 1, 1e-3, 0.9, 0.999, 1e-15)),
               dict(group=_lib.AdamGroup(1024, 0, 1024, 1024, 8, 1, 1e-3, 0.9, 0.999, 1e-15))):
        assert step(**kw) == -1, kw
    assert step(nbytes=8) == -3


def test_refusals():
    from pogs_amd.dist import ShardAdam
    from pogs_amd.optim import clip_grad_norm_, grad_norm

    g = torch.ones(4)
    with pytest.raises(RuntimeError, match="HIP device"):
        grad_norm([g])
    with pytest.raises(RuntimeError, match="HIP device"):
        clip_grad_norm_(_params([g]), 1.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_(_params([g]), bad)
    for bad in (3.0, 0.0, -math.inf):
        with pytest.raises(ValueError, match="norm_type"):
            clip_grad_norm_(_params([g]), 1.0, norm_type=bad)
        with pytest.raises(ValueError, match="norm_type"):
            grad_norm([g], bad)
    # nothing to clip: torch's answer
    assert grad_norm([]).item() == 0.0 and clip_grad_norm_([], 1.0).item() == 0.0
    assert clip_grad_norm_([torch.zeros(3, requires_grad=True)], 1.0).item() == 0.0
    with pytest.raises(ValueError, match="max_norm"):
        ShardAdam({"a": {"lr": 1e-3, "max_norm": 1.0}})
    ShardAdam({"a": {"lr": 1e-3, "max_norm": None}})


class _OnADevice:
    """As much of a parameter with a gradient as the optimiser looks at before it touches anything."""

    is_cuda, dtype, grad = True, torch.float32, torch.ones(4)

    def __init__(self, device):
        self.device = device

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.device


def test_clipped_steps_are_refused_before_they_begin():
    from pogs_amd.optim import Optimizers

    p, q, r = _OnADevice(0), _OnADevice(0), _OnADevice(1)
    clip = {"lr": 1e-3, "max_norm": 1.0}

    def refused(opt, error, match, names, **kw):
        with pytest.raises(error, match=match):
            opt.optimizer_step_some(names, **kw)
        assert all(opt.state(name, i) == {} for name in opt.parameters for i in range(len(opt.parameters[name])))

    opt = Optimizers({"a": dict(clip), "b": dict(clip), "c": {"lr": 1e-3}}, {"a": [p], "b": [p, q], "c": [r]})
    refused(opt, ValueError, "twice", ["a", "a"])
    refused(opt, ValueError, "twice", ["a", "b"])
    refused(opt, RuntimeError, "one device", ["a", "c"])
    free = Optimizers({"a": {"lr": 1e-3}, "b": {"lr": 1e-3}}, {"a": [p, p], "b": [q, r]})
    refused(free, ValueError, "twice", ["a"], max_norm=1.0)
    refused(free, RuntimeError, "one device", ["b"], max_norm=1.0)
    for bad in (-1.0, math.nan):                # set after the optimiser was made
        opt.config["a"]["max_norm"] = bad
        refused(opt, ValueError, "max_norm", ["a"])


def test_one_block_recognises_dense_layouts():
    from pogs_amd.optim import _one_block

    a = torch.zeros(4, 6, 5)
    assert _one_block(a) and _one_block(a.permute(2, 0, 1)) and _one_block(a[:, :1, :1].transpose(0, 1)[:, :1])
    assert _one_block(torch.zeros(3, 1, 2).expand(3, 1, 2)) and _one_block(torch.zeros(()))
    assert not _one_block(a[:, ::2]) and not _one_block(a[:, :, :4]) and not _one_block(torch.zeros(3, 1).expand(3, 5))


# ---- on the GPU -------------------------------------------------------------------------------------------------------
SIZES = {
    "one value": [1],
    "ragged": [1, 3, 4, 5, 63, 64, 65, 4095, 8191, 8192, 8193, 100_003],
    "many": [1 + 37 * i for i in range(300)],          # more than one launch's table
    "large": [9_000_001, 17, 4_000_000],
    "empty among": [0, 5, 0, 70_000, 0],
}


def _grads(sizes, dtypes, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=gen) * scale * (1 + i % 5)).to(dtypes[i % len(dtypes)]).cuda()
            for i, n in enumerate(sizes)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float16,),
                                    (torch.float32, torch.bfloat16, torch.float16)], ids=["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("which", list(SIZES))
def test_norm_and_clip(which, dtypes, kind):
    from pogs_amd.optim import clip_grad_norm_, grad_norm

    grads = _grads(SIZES[which], dtypes, seed=len(which))
    want = _norm64(grads, kind)
    norm = grad_norm(grads, kind)
    assert norm.dtype == torch.float32 and norm.dim() == 0 and norm.is_cuda
    assert abs(norm.item() - want) <= (U + 2.0 ** -40) * want
    assert torch.equal(norm, grad_norm(grads, kind))
    before = [g.cpu().double() for g in grads]
    params = _params(grads)
    # within bounds: untouched
    got = clip_grad_norm_(params, want * 1.01, kind)
    assert torch.equal(got, norm)
    assert all(torch.equal(p.grad.cpu().double(), b) for p, b in zip(params, before))
    limit = 0.3 * want
    got = clip_grad_norm_(params, limit, kind)
    assert torch.equal(got, norm)
    c = limit / (want + 1e-6)
    for p, b in zip(params, before):
        half = HALF_STEP[p.grad.dtype]
        bound = b.abs() * c * (4 * U + (half if half != U else 0.0)) * 1.001
        if p.grad.dtype == torch.float16:
            bound = bound + 2.0 ** -25        # below the normal range a half step is absolute
        assert ((p.grad.cpu().double() - b * c).abs() <= bound).all()


@pytest.mark.gpu
def test_views_of_one_buffer_layouts_and_strides():
    """Gradients that are odd offsets into one flat buffer (each view of its own alignment), transposed, and strided;
    what lies between and behind them stays as it was."""
    from pogs_amd.optim import clip_grad_norm_, grad_norm

    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        gen = torch.Generator().manual_seed(2)
        flat = torch.randn(60_000, generator=gen).to(dtype).cuda()
        copy = flat.clone()
        views = [flat[1:4], flat[5:9002], flat[9002:20_003], flat[20_010:50_010].view(100, 300).t(),
                 flat[50_010:58_010].view(40, 200)[:, ::3]]
        held = torch.zeros(60_000, dtype=torch.bool)
        for v in views:
            held.as_strided(v.shape, v.stride(), v.storage_offset()).fill_(True)
        want = _norm64(views, 2)
        assert abs(grad_norm(views).item() - want) <= (U + 2.0 ** -40) * want
        clip_grad_norm_(_params(views), 0.5 * want)
        got, src = flat.cpu().double(), copy.cpu().double()
        assert torch.equal(got[~held], src[~held])
        half = HALF_STEP[dtype] + 4 * U
        assert ((got - 0.5 * src)[held].abs() <= half * 1.01 * 0.5 * src[held].abs() + 2.0 ** -24).all()
    # an expanded gradient has a norm, over all its elements, but cannot be scaled in place
    e = torch.full((1, 3), 2.0, device="cuda").expand(4, 3)
    assert grad_norm([e]).item() == pytest.approx(math.sqrt(48), rel=2 * U)


@pytest.mark.gpu
def test_a_scattered_gradient_listed_twice_is_refused():
    from pogs_amd.optim import clip_grad_norm_

    p = torch.zeros(6, 4, device="cuda", requires_grad=True)
    p.grad = torch.ones(6, 8, device="cuda")[:, ::2]
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_([p, p], 1.0)
    assert float(p.grad.min()) == 1.0
    assert clip_grad_norm_([p], 1.0).item() == pytest.approx(math.sqrt(24), rel=2 * U)


@pytest.mark.gpu
def test_autograd_notices_that_gradients_were_scaled():
    from pogs_amd.optim import clip_grad_norm_

    p = torch.ones(100, device="cuda", requires_grad=True)
    p.grad = torch.full((100,), 3.0, device="cuda")
    q = torch.ones(100, device="cuda", requires_grad=True)
    loss = (q * p.grad).sum()
    clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
def test_gradients_without_elements():
    from pogs_amd.optim import Optimizers, clip_grad_norm_, grad_norm

    for dtype in (torch.float32, torch.bfloat16):
        p = _params([torch.zeros(0, 3, device="cuda", dtype=dtype), torch.zeros(0, device="cuda", dtype=dtype)])
        torch.full((4096,), 7.0, device="cuda")                # what the norm's memory may have held before
        assert clip_grad_norm_(p, 1.0).item() == 0.0
        assert grad_norm([q.grad for q in p]).item() == 0.0
    q = {"a": [torch.zeros(0, device="cuda", requires_grad=True)], "b": [torch.ones(5, device="cuda", requires_grad=True)]}
    q["a"][0].grad, q["b"][0].grad = torch.zeros(0, device="cuda"), torch.full((5,), 2.0, device="cuda")
    opt = Optimizers({k: {"lr": 0.5, "max_norm": 1.0} for k in q}, q)
    opt.optimizer_step_all()
    assert opt.grad_norms["a"].item() == 0.0 and opt.grad_norms["b"].item() == pytest.approx(math.sqrt(20), rel=2 * U)
    assert ((q["b"][0] - 0.5).abs() <= 8 * U).all()            # a first step moves by the rate


@pytest.mark.gpu
def test_extreme_values_and_what_is_not_finite():
    from pogs_amd.optim import clip_grad_norm_, grad_norm

    big = torch.full((1000,), 1e30, device="cuda")
    assert grad_norm([big]).item() == pytest.approx(1e30 * math.sqrt(1000), rel=4 * U)      # squares pass float32's range
    tiny = torch.full((1000,), 1e-38, device="cuda")
    assert grad_norm([tiny]).item() == pytest.approx(1e-38 * math.sqrt(1000), rel=1e-6)
    zero = torch.zeros(77, device="cuda")
    p = _params([zero])
    assert clip_grad_norm_(p, 0.0).item() == 0.0 and torch.equal(p[0].grad, zero)
    a = torch.ones(500, device="cuda")
    b = torch.ones(500, device="cuda", dtype=torch.bfloat16)
    a[3] = math.nan
    for kind in (1.0, 2.0, math.inf):
        assert math.isnan(grad_norm([b, a], kind).item())
    p = _params([a, b])
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
    assert torch.isfinite(b).all()
    assert math.isnan(clip_grad_norm_(p, 1.0).item())
    assert torch.isnan(p[0].grad).all() and torch.isnan(p[1].grad).all()
    a = torch.ones(500, device="cuda")
    a[7] = -math.inf
    p = _params([a])
    assert clip_grad_norm_(p, 1.0).item() == math.inf
    assert math.isnan(p[0].grad[7].item()) and float(p[0].grad[:7].abs().max()) == 0.0
    assert math.isnan(grad_norm([torch.tensor([math.inf, math.nan], device="cuda")], math.inf).item())


@pytest.mark.gpu
def test_refused_on_the_device():
    from pogs_amd.optim import Optimizers, clip_grad_norm_

    p = _params([torch.ones(100, device="cuda")])
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_(p + p, 1.0)
    assert float(p[0].grad.min()) == 1.0
    with pytest.raises(TypeError, match="float64"):
        clip_grad_norm_(_params([torch.ones(3, device="cuda", dtype=torch.float64)]), 1.0)
    q = torch.zeros(4, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="max_norm"):
        Optimizers({"a": {"lr": 1e-3, "max_norm": -1.0}}, {"a": [q]})
    opt = Optimizers({"a": {"lr": 1e-3, "max_norm": 1.0}}, {"a": [q]})
    with pytest.raises(ValueError, match="exclude"):
        opt.optimizer_step_all(max_norm=1.0)
    opt.optimizer_step_all()                    # no gradient anywhere: nothing happens
    assert opt.grad_norms == {} and opt.state("a") == {}


def _adam64(p, g, st, lr, limit, norm):
    c = 1.0 if limit is None else min(1.0, limit / (norm + 1e-6))
    g = g * c
    st["t"] += 1
    st["m"] = 0.9 * st["m"] + 0.1 * g
    st["v"] = 0.999 * st["v"] + 0.001 * g * g
    return p - lr * (st["m"] / (1 - 0.9 ** st["t"])) / ((st["v"] / (1 - 0.999 ** st["t"])).sqrt() + 1e-15)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["per group", "over all", "some groups", "more groups than a launch takes"])
def test_clipped_adam(mode):
    from pogs_amd.optim import Optimizers

    sizes = {"a": [5, 4097], "b": [64 * 1001], "c": [3, 1, 33]}
    if mode.startswith("more"):
        sizes = {"g%d" % i: [7 + i, 3] for i in range(40)}
    own = {"per group": sizes, "some groups": ["b"], "over all": []}.get(mode, sizes)
    gen = torch.Generator().manual_seed(9)
    params = {k: [torch.randn(n, generator=gen) for n in v] for k, v in sizes.items()}
    limits = {k: 0.2 + 0.1 * i for i, k in enumerate(sizes)}
    dev = {k: [p.cuda().requires_grad_(True) for p in v] for k, v in params.items()}
    opt = Optimizers({k: {"lr": 0.01, "max_norm": limits[k] if k in own else None} for k in sizes}, dev)
    ref = {k: [p.double() for p in v] for k, v in params.items()}
    st = {k: [dict(t=0, m=torch.zeros_like(p), v=torch.zeros_like(p)) for p in v] for k, v in ref.items()}
    for step in range(4):
        grads = {k: [torch.randn(n, generator=gen) * (0.01 if step == 2 else 1.0) for n in v] for k, v in sizes.items()}
        for k, v in dev.items():
            for p, g in zip(v, grads[k]):
                p.grad = g.cuda()
        total = _norm64([g for v in grads.values() for g in v], 2)
        if mode == "over all":
            opt.optimizer_step_all(max_norm=1.5)
        else:
            opt.optimizer_step_all()
        assert set(opt.grad_norms) == set(sizes if mode == "over all" else own)
        for k in sizes:
            norm = total if mode == "over all" else _norm64(grads[k], 2)
            limit = 1.5 if mode == "over all" else (limits[k] if k in own else None)
            if limit is not None:
                assert abs(opt.grad_norms[k].item() - norm) <= 2 * U * norm
            for i, g in enumerate(grads[k]):
                assert torch.equal(dev[k][i].grad.cpu(), g)      # gradients keep their values
                old = {x: st[k][i][x].clone() for x in "mv"}
                ref[k][i] = _adam64(ref[k][i], g.double(), st[k][i], 0.01, limit, norm)
                got = opt.state(k, i)
                c = 1.0 if limit is None else min(1.0, limit / (norm + 1e-6))
                top = torch.maximum(old["m"].abs(), g.double().abs() * c)
                # errors of earlier steps come in through the old moments, at most once each
                assert ((got["exp_avg"].cpu().double() - st[k][i]["m"]).abs() <= 8 * U * (step + 1) * top.max()).all()
                top = torch.maximum(old["v"], (g.double() * c) ** 2)
                assert ((got["exp_avg_sq"].cpu().double() - st[k][i]["v"]).abs() <= 16 * U * (step + 1) * top.max()).all()
    # the step is 0.01 times a quotient of at most about one whose two sides carry the errors above relative to the
    # largest entry; an entry far below it can be off by more, so the parameters are held in the 2-norm
    for k in sizes:
        for p, r in zip(dev[k], ref[k]):
            off = (p.detach().cpu().double() - r).norm().item()
            assert off <= (8 * U * r.norm().item() + 4 * 0.01 * 64 * U * math.sqrt(r.numel())), k


@pytest.mark.gpu
def test_clipping_in_a_graph_and_on_another_stream():
    from pogs_amd.optim import Optimizers, clip_grad_norm_

    grads = _grads([100_003, 777, 64], (torch.float32, torch.bfloat16), seed=4)
    params = _params([g.clone() for g in grads])
    opt_p = [torch.randn(70_001, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_(True)]
    opt_p[0].grad = torch.randn(70_001, device="cuda")
    opt = Optimizers({"a": {"lr": 0.0, "max_norm": 1.0}}, {"a": opt_p})
    opt.optimizer_step_all()                       # state exists before the capture

    def eager(src):
        ps = _params([g.clone() for g in src])
        n = clip_grad_norm_(ps, 2.0)
        return n, [p.grad for p in ps]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n0, g0 = eager(grads)
    torch.cuda.current_stream().wait_stream(side)
    n1, g1 = eager(grads)
    assert torch.equal(n0, n1) and all(torch.equal(a, b) for a, b in zip(g0, g1))
    graphs = []
    for limit in (2.0, 1.0):                       # two graphs that live together
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = clip_grad_norm_(params, limit)
            opt.optimizer_step_all()
            step_norm = opt.grad_norms["a"]
        graphs.append((graph, norm, step_norm, limit))
    for i in range(3):
        for graph, norm, step_norm, limit in graphs:
            fresh = _grads([100_003, 777, 64], (torch.float32, torch.bfloat16), seed=10 + i)
            for p, g in zip(params, fresh):
                p.grad.copy_(g)
            opt_p[0].grad.mul_(1.5)
            graph.replay()
            junk = torch.full((1 << 20,), 3.0, device="cuda").sum()      # eager work between the replays
            ps = _params(fresh)
            want = clip_grad_norm_(ps, limit)
            assert torch.equal(norm, want)
            assert all(torch.equal(p.grad, q.grad) for p, q in zip(params, ps))
            w = _norm64([opt_p[0].grad], 2)
            assert abs(step_norm.item() - w) <= 2 * U * w
            del junk


@pytest.mark.gpu
def test_matches_torch_clip_grad_norm():
    """The reference's own function on the same gradients; torch sums in float32, the tolerance is its share."""
    from pogs_amd.optim import clip_grad_norm_

    grads = _grads([3000, 45_000, 1000, 64_000], (torch.float32,), seed=8)
    a, b = _params([g.clone() for g in grads]), _params([g.clone() for g in grads])
    n = clip_grad_norm_(a, 1.0)
    m = torch.nn.utils.clip_grad_norm_(b, 1.0)
    assert abs(n.item() - m.item()) <= 1e-6 * m.item()
    for x, y in zip(a, b):
        assert ((x.grad - y.grad).abs() <= 2e-6 * y.grad.abs()).all()


def test_clipped_steps_of_an_iterator_are_refused_before_they_begin():
    from pogs_amd.optim import Optimizers

    p = _OnADevice(0)
    free = Optimizers({"a": {"lr": 1e-3}}, {"a": [p, p]})
    with pytest.raises(ValueError, match="twice"):
        free.optimizer_step_some(iter(["a"]), max_norm=1.0)


@pytest.mark.gpu
def test_an_expanded_gradient_is_refused_before_anything_is_scaled(gpu):
    from pogs_amd.optim import clip_grad_norm_, grad_norm

    p, q = torch.zeros(64, device=gpu, requires_grad=True), torch.zeros(8, 4, device=gpu, requires_grad=True)
    p.grad, q.grad = torch.ones(64, device=gpu), torch.ones(8, 1, device=gpu).expand(8, 4)
    with pytest.raises(RuntimeError, match="expanded"):
        clip_grad_norm_([p, q], 0.5)
    assert (p.grad == 1).all() and (q.grad == 1).all()
    assert grad_norm([p.grad, q.grad]).item() == pytest.approx(96 ** 0.5, rel=1e-6)
    one = torch.zeros(1, 6, device=gpu, requires_grad=True)       # of one row only: nothing is written twice
    one.grad = torch.ones(12, device=gpu).as_strided((1, 6), (0, 2))
    assert clip_grad_norm_([p, one], 0.5).item() == pytest.approx(70 ** 0.5, rel=1e-6)
    assert torch.equal(one.grad[0], p.grad[:6]) and (p.grad < 0.1).all()
