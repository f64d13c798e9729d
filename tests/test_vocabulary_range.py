"""Vocabulary cross entropy where rows, words or upstream gradients differ by many orders of magnitude: every output is held
to a bound from its own row's or word's magnitudes, not from the tensor's largest.

With u = 2^-24 (half a float32 step), for float32 input tau = 3 * 2^-22 (a value is kept in 22 bits, and so is the product of
two) and for 16-bit input 0:
  logits     dz = |scale| (tau + (n D / 16 + 16) u) sum_d |x_d w_d|: D products added 16 at a time in n passes (n at most 6),
             and for float32 2^-36 of the row's largest times the word's largest a feature (what 22 bits of two planes leave
             out of values far below their row's largest)
  log-sum    the largest dz that counts, (104 + words / 4096) u and 8 u |lse|
  G          a p times (dz + dlse + 8 u (|z| + |lse|) in the exponent) + 16 u a p + 8 u b at the label + the pieces it is kept in:
             2^-15 |G| (16-bit input), 2^-21 |G| (float32)
  gradients  scale sum |dG| |m| + scale (tau + (n K / 16 + 24) u) sum |G| |m| over the axis of K that is added up (float32: the
             planes' 2^-36 of the largest of a row m as well) + half a step of the output's type
  underflow  2^-120 of the largest coefficient, G and m.
"""
import math

import pytest
import torch

U = 2.0 ** -24
HALF = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
PASSES = 6
IGN = -100


def reference(x, w, labels, scale, up, ignore=IGN, exact=False):
    """Values and bounds in float64: loss, lse, dx and dw; up: the rows' upstream gradients of the loss.  exact: every sum of
    a logit is a float32 number, so that only the scale rounds it."""
    dtype, (P, D), V = x.dtype, x.shape, w.shape[0]
    tau = 3 * 2.0 ** -22 if dtype == torch.float32 else 0.0
    held = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -15
    keep = labels != ignore
    x = torch.where(keep[:, None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device))
    w, up = w.double(), up.double() * keep
    at = torch.where(keep, labels, torch.zeros_like(labels))[:, None]
    z = scale * torch.mm(x, w.t().contiguous())
    planes = 2.0 ** -36 if dtype == torch.float32 else 0.0
    xmax, wmax = x.abs().amax(1), w.abs().amax(1)
    dz = abs(scale) * (torch.mm(x.abs(), w.abs().t().contiguous()) * (tau + (PASSES * D / 16 + 16) * U)
                       + planes * D * xmax[:, None] * wmax)
    if exact:
        dz = 4 * U * z.abs()
    lse = torch.logsumexp(z, 1)
    p = (z - lse[:, None]).exp()
    # a word's logit counts in the log-sum as far as it is probable
    dlse = (p * dz).sum(1) * 1.01 + (104 + V / 4096) * U + 8 * U * lse.abs()
    zt = z.gather(1, at)[:, 0]
    out = {"lse": (lse * keep, dlse * keep),
           "loss": ((lse - zt) * keep, (dlse + dz.gather(1, at)[:, 0] + 8 * U * (lse.abs() + zt.abs())) * keep)}
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    a = up.abs()[:, None]
    G = up[:, None] * (p - hot)
    dG = (a * p * ((dz + dlse[:, None] + 8 * U * (z.abs() + lse.abs()[:, None])) * 1.01 + 16 * U) + 8 * U * a * hot + held * G.abs()
          + 2.0 ** -120 * a.max())

    def grad(G, dG, m):
        v = scale * torch.mm(G, m)
        e = abs(scale) * (torch.mm(dG, m.abs()) + torch.mm(G.abs(), m.abs()) * (tau + (PASSES * G.shape[1] / 16 + 24) * U)
                          + planes * torch.mm(G.abs(), m.abs().amax(1, keepdim=True)) + 2.0 ** -120 * G.abs().max() * m.abs().max())
        return v, e * 1.01 + HALF[dtype] * v.abs() * 1.01 + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -140)

    out["dx"], out["dw"] = grad(G, dG, w), grad(G.t().contiguous(), dG.t().contiguous(), x)
    return out


def close(got, want, what, tight=0.5, rows=None):
    """Every element within its bound, and the bound below a tenth of the value for a share `tight` of the elements, so that
    it could not hold for any result."""
    value, bound = want
    assert got.shape == value.shape, what
    # (a value beyond the type's range, as of a float16 gradient of 1e4 times a feature of 8, has no finite result)
    rows = (value.abs() + bound <= torch.finfo(got.dtype).max) & (True if rows is None else rows)
    got, value, bound = got.detach().double()[rows], value[rows], bound[rows]
    assert torch.isfinite(got).all(), what
    off = (got - value).abs() - bound
    worst = off.argmax()
    assert off.max() <= 0, (what, worst.item(), got.reshape(-1)[worst].item(), value.reshape(-1)[worst].item(),
                            bound.reshape(-1)[worst].item())
    share = (bound <= 0.1 * value.abs()).double().mean().item()
    assert share >= tight, (what, "bound too wide", share)


def run(x, w, labels, scale, up):
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss, lse = vocabulary_cross_entropy(x, w, labels, scale, reduction="none", return_lse=True)
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    return {"loss": loss, "lse": lse, "dx": dx, "dw": dw}


def inputs(P, V, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g) / D ** 0.5
    labels = torch.randint(0, V, (P,), generator=g)
    x = torch.randn(P, D, generator=g) + w[labels]
    return x.to(dtype).cuda(), w.to(dtype).cuda(), labels.cuda(), g


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("P,V,D", [(300, 1000, 64), (513, 700, 130), (20, 6000, 130), (50, 6000, 96), (100, 6000, 128)])
def test_rows_of_very_different_weight(P, V, D, dtype):
    """Rows weighted over eight decades: the gradient of a row with a small weight is as good as that of a large one."""
    x, w, y, g = inputs(P, V, D, dtype, seed=P)
    weight = torch.logspace(4, -4, P)[torch.randperm(P, generator=g)].cuda()
    if dtype == torch.float32:
        weight = weight * 1e-4
    ref = reference(x, w, y, 2.0, weight)
    got = run(x, w, y, 2.0, weight)
    for k in ("loss", "lse", "dx", "dw"):
        close(got[k], ref[k], k)


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("P,V,D", [(300, 1000, 512), (100, 2000, 512)])
def test_words_that_are_nobodys_label(P, V, D, dtype):
    """Sharp logits: the words without a label have probabilities down to 1e-38, and their gradients are small, not zero."""
    x, w, y, g = inputs(P, V, D, torch.float32, seed=5)
    y = y % 200
    w = w / w.norm(dim=1, keepdim=True)
    x = w[y] + 0.02 * torch.randn(P, D, generator=g).cuda()
    x, w = (x / x.norm(dim=1, keepdim=True)).to(dtype), w.to(dtype)
    for scale in (10.0, 30.0, 100.0):
        up = torch.full((P,), 2.0 ** 9 if dtype == torch.float16 else 1.0 / P, device="cuda")
        ref = reference(x, w, y, scale, up)
        got = run(x, w, y, scale, up)
        for k in ("lse", "dw"):
            # (float16 holds gradients down to 2^-24; at 100 many of these are near the smallest of float32)
            close(got[k], ref[k], k, tight=0.0 if scale > 50 or (dtype == torch.float16 and scale > 20) else 0.4)
        # (a single element may be below the smallest float32)
        assert dtype == torch.float16 or (got["dw"][200:] != 0).any(dim=1).all()


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("P,V,D", [(300, 700, 40), (129, 64, 16), (20, 9000, 64), (100, 9000, 64), (20, 40_000, 16),
                                   (100, 40_000, 16)])
@pytest.mark.parametrize("exponent", [6, 20, 30, 60])
def test_logits_far_beyond_the_differences_that_float32_holds(P, V, D, exponent, dtype):
    """Small whole numbers and a power of two as scale: logits are exact, and equal ones have to stay equal.  A probability is
    1 / ties for the largest and (from 2^6 on, below 2^-92) nothing for the others."""
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    g = torch.Generator().manual_seed(exponent)
    x = torch.randint(-3, 4, (P, D), generator=g).to(dtype).cuda()
    w = torch.randint(-3, 4, (V, D), generator=g).to(dtype).cuda()
    y = torch.randint(0, V, (P,), generator=g).cuda()
    up = torch.randint(1, 5, (P,), generator=g).float().cuda() * 2.0 ** -exponent
    scale = 2.0 ** exponent
    z = torch.mm(x.double(), w.double().t().contiguous())
    best = z == z.amax(1, keepdim=True)
    p = best / best.sum(1, keepdim=True)
    lse = scale * z.amax(1) + best.sum(1).double().log()
    zt = scale * z.gather(1, y[:, None])[:, 0]
    G = up.double()[:, None] * (p - torch.zeros_like(p).scatter_(1, y[:, None], 1.0))
    held = 2.0 ** -20 if dtype == torch.float32 else 2.0 ** -14
    with torch.no_grad():
        plain, plain_lse = vocabulary_cross_entropy(x, w, y, scale, reduction="none", return_lse=True)
    got = run(x, w, y, scale, up)
    # a logarithm to base 2 and back: two roundings of the logit and one of the result
    for loss, s in ((got["loss"], got["lse"]), (plain, plain_lse)):
        close(s, (lse, 8 * U * lse.abs() + 16 * U), "lse")
        close(loss, (lse - zt, 8 * U * (lse.abs() + zt.abs()) + 16 * U), "loss")
    for k, gr, m in (("dx", G, w), ("dw", G.t().contiguous(), x)):
        v = scale * torch.mm(gr, m.double())
        bound = scale * torch.mm(gr.abs(), m.double().abs()) * held + HALF[dtype] * 1.01 * v.abs() + 2.0 ** -80
        close(got[k], (v, bound), k, tight=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("P,V,D", [(300, 1000, 64), (257, 333, 136), (140, 700, 512), (100, 9000, 64)])
@pytest.mark.parametrize("exponent", [40, -40, 90])
@pytest.mark.parametrize("which", ["row", "word"])
def test_one_row_or_word_of_another_magnitude(P, V, D, exponent, which, dtype):
    """A row (or word) 2^40 or 2^90 times as large as the others, or as small, counts as one row (word): the others keep
    their values."""
    x, w, y, g = inputs(P, V, D, dtype, seed=P + exponent)
    odd = 37
    t = x if which == "row" else w
    t[odd] = (t[odd].double() * 2.0 ** exponent).to(dtype)
    up = torch.randn(P, generator=g).cuda()
    ref = reference(x, w, y, 2.0, up)
    got = run(x, w, y, 2.0, up)
    z = 2.0 * torch.mm(x.double(), w.double().t().contiguous())
    others = (z.abs() < 1e4).all(dim=1) if which == "row" else z[:, odd] < 1e3    # rows that do not take the odd word alone
    assert others.sum() > P // 3
    for k in ("loss", "lse", "dx"):
        close(got[k], ref[k], k, rows=others if got[k].dim() == 1 else others[:, None])
    words = torch.ones(V, dtype=torch.bool, device="cuda")
    if exponent > 0 and which == "row":           # the words that the odd row moves hold its gradient, of its size
        words[y[odd]] = words[z[odd].argmax()] = False
    elif exponent > 0:
        words[odd] = False
    close(got["dw"], ref["dw"], "dw", rows=words[:, None], tight=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("P,V,D", [(300, 1000, 64), (130, 500, 33), (1025, 400, 8)])
@pytest.mark.parametrize("which", ["rows", "words"])
def test_rows_or_words_over_many_powers_of_two(P, V, D, which):
    x, w, y, g = inputs(P, V, D, torch.float32, seed=P)
    t = x if which == "rows" else w
    t *= (2.0 ** torch.randint(-60, 1, (len(t),), generator=g).double()).float().cuda()[:, None]
    up = torch.ones(P, device="cuda")
    ref = reference(x, w, y, 3.0, up)
    got = run(x, w, y, 3.0, up)
    for k in ("loss", "lse", "dx", "dw"):
        close(got[k], ref[k], k)


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """A tangent would be dropped, and read as a derivative of zero."""
    import torch.autograd.forward_ad as fwd

    from pogs_amd.optim import grad_norm
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, y = torch.randn(4, 8), torch.randn(5, 8), torch.zeros(4, dtype=torch.int64)
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        dual = fwd.make_dual(x, torch.ones_like(x))
        for args in ((dual, w, y), (dual * 2, w, y), (x, fwd.make_dual(w, w), y)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                vocabulary_cross_entropy(*args)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            grad_norm([x, dual])
        with pytest.raises(RuntimeError, match="HIP device"):     # a level that no tensor takes part in is none
            vocabulary_cross_entropy(x, w, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("P,V,D,exp_x,exp_w", [(P, V, D, *e) for P, V, D in ((200, 300, 64), (300, 5000, 64))
                                               for e in ((-60, -60), (0, -100), (-100, 0), (-100, 4), (40, 60))]
                         + [(40, 20_000, 32, *e) for e in ((-40, -40), (0, -80), (-80, 0), (40, 60))])
def test_a_scale_near_the_ends_of_float32(P, V, D, exp_x, exp_w, dtype):
    """Powers of two that cancel in the logits: the same bits as without them, in the gradients too."""
    x, w, y, g = inputs(P, V, D, dtype, seed=P)
    up = torch.randn(P, generator=g).cuda()
    base = run(x, w, y, 1.0, up)
    got = run(x * 2.0 ** exp_x, w * 2.0 ** exp_w, y, 2.0 ** -(exp_x + exp_w), up)
    for k, e in (("loss", 0), ("lse", 0), ("dx", exp_x), ("dw", exp_w)):
        # (values that the scale takes below the smallest float32 are left out)
        want, have = base[k].double(), got[k].double() * 2.0 ** e
        held = (base[k].double() * 2.0 ** -e).abs() > 2.0 ** -125
        assert torch.isfinite(got[k]).all() and torch.equal(have[held], want[held]), k


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("P", [4096, 4097, 9001])
def test_many_rows_of_very_different_weight(P, dtype):
    """More rows than one workgroup makes the factors of; the largest is in the last one's."""
    x, w, y, g = inputs(P, 300, 32, dtype, seed=P)
    weight = torch.logspace(-4, 3, P).cuda() * (1e-4 if dtype == torch.float32 else 1.0)
    ref = reference(x, w, y, 2.0, weight)
    got = run(x, w, y, 2.0, weight)
    for k in ("loss", "lse", "dx", "dw"):
        close(got[k], ref[k], k, tight=0.2 if k == "dw" else 0.5)


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("P,V,D", [(17, 3, 700_001), (2, 3, 1_040_000), (129, 5, 60_003)])
@pytest.mark.parametrize("sparse", ["features", "vocabulary"])
def test_many_features(P, V, D, sparse, dtype):
    """Eighths of small whole numbers, and zeros but for some 300 columns in one of the factors: logits are exact in any
    order of their sum, so the width of the rows leaves no room in the bounds, and the other factor fills every column of
    the gradient that is made of it."""
    g = torch.Generator().manual_seed(P)
    x, w = (torch.randint(1, 4, (n, D), generator=g) * (2 * torch.randint(0, 2, (n, D), generator=g) - 1) / 8.0 for n in (P, V))
    edges = [0, 1, 7, 8, 31, 32, 63, 64, 255, 256, 511, 512, 4095, 4096, 65535 % D, D // 2, D - 257, D - 65, D - 33, D - 9, D - 2, D - 1]
    keep = torch.zeros(D)
    keep[torch.cat([torch.tensor(edges), torch.randint(0, D, (280,), generator=g)])] = 1.0
    if sparse == "features":
        x = x * keep
    else:
        w = w * keep
    x, w = x.to(dtype).cuda(), w.to(dtype).cuda()
    y = torch.randint(0, V, (P,), generator=g).cuda()
    up = torch.randn(P, generator=g).cuda()
    ref = reference(x, w, y, 0.25, up, exact=True)
    got = run(x, w, y, 0.25, up)
    for k in ("loss", "lse", "dx", "dw"):
        close(got[k], ref[k], k, tight=0.0 if sparse == {"dx": "vocabulary", "dw": "features"}.get(k) else 0.9)
    # nothing reaches a column in which the other factor is zero
    none = keep.cuda() == 0
    assert (got["dw" if sparse == "features" else "dx"][:, none] == 0).all()
