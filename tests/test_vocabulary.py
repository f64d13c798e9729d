"""Cross entropy over a vocabulary of embeddings (pr_vocab_ce_*, pogs_amd.vocabulary) against the formulas in float64.

Tolerances, element by element, from u = 2^-24 (half a float32 step) and the operands' rounding:
  logits     a 16-bit operand is exact in float16 planes; a float32 one loses 2^-22, and so does leaving out the product
             of the residuals: rho = 0 or 3 * 2^-22 of sum_d |x_d w_d|.  Adding D products in float32, 16 at a time, n_p
             passes (1 or 3): (n_p D / 16 + 16) u of the same sum.  Values 2^-38 below the tensor's largest are lost.
  log-sum    the largest logit error, the exponentials' sums (at most 64 + 32 + pairs / 32 terms after one another) and
             the roundings of maximum and logarithm, 8 u |lse|
  G          a p (the errors of logit and log-sum, 8 u of their size for the exponent) + the rounding to float16
             (2^-11 of G; two planes: 3 * 2^-22) + what underflows, 2^-36 of the largest coefficient
  gradients  scale |dG| |w| summed, the additions as above over the long axis, the operand's rounding and half a step of
             the output's type (float16 below its normal range: 2^-25)."""
import ctypes
import math

import pytest
import torch

from pogs_amd import _lib

U = 2.0 ** -24
NP = {torch.float32: 2, torch.float16: 1, torch.bfloat16: 1}
HALF = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
IGN = -100


def reference(x, w, labels, scale, g_loss, g_lse, ignore=IGN, dtype=None, n3=None):
    """Values and bounds in float64; g_loss, g_lse: [P] gradients of the row losses and of the log-sums."""
    dtype = dtype or x.dtype
    n3 = n3 or (3 if NP[dtype] == 2 else 1)
    rho = 3 * 2.0 ** -22 if NP[dtype] == 2 else 0.0
    P, D = x.shape
    V = w.shape[0]
    keep = labels != ignore
    x, w = x.double() * keep[:, None], w.double()
    x = torch.where(keep[:, None], x, torch.zeros_like(x))
    at = torch.where(keep, labels, torch.zeros_like(labels))
    z = scale * (x @ w.t())
    mag = x.abs() @ w.abs().t() + 2.0 ** -38 * D * x.abs().max() * w.abs().max()
    dz = abs(scale) * mag * (rho + (n3 * D / 16 + 16) * U)
    lse = torch.logsumexp(z, 1)
    pairs = (V + 255) // 256 * 2
    dlse = dz.amax(1) + (104 + pairs / 32) * U + 8 * U * lse.abs()
    zt = z.gather(1, at[:, None])[:, 0]
    out = {"loss": ((lse - zt) * keep, (dlse + dz.gather(1, at[:, None])[:, 0] + 8 * U * (lse.abs() + zt.abs())) * keep),
           "lse": (lse * keep, dlse * keep)}
    b = g_loss * keep
    a = b + g_lse * keep
    p = (z - lse[:, None]).exp()
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    G = a[:, None] * p - b[:, None] * hot
    top = torch.maximum(a.abs(), b.abs()).max() if P else torch.zeros(())
    half_g = 2.0 ** -11 if NP[dtype] == 1 else 3 * 2.0 ** -22
    dG = (a[:, None].abs() * p * ((dz + dlse[:, None] + 8 * U * (z.abs() + lse[:, None].abs())) * 1.01 + 16 * U)
          + 8 * U * (a.abs() + b.abs())[:, None] * (p + hot) + G.abs() * half_g + 2.0 ** -36 * top)
    dG = dG * keep[:, None]

    def grad(G, dG, m):
        v = scale * (G @ m)
        e = abs(scale) * (dG @ m.abs() + (G.abs() @ m.abs()) * (rho + (n3 * G.shape[1] / 16 + 24) * U)
                          + G.abs().sum(1, keepdim=True) * 2.0 ** -38 * m.abs().max())
        return v, e * 1.01 + HALF[dtype] * v.abs() * 1.01 + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -140)

    out["dx"], out["dw"] = grad(G, dG, w), grad(G.t().contiguous(), dG.t().contiguous(), x)
    return out


def close(got, want, what):
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape, what
    assert torch.isfinite(got).all(), what
    off = (got - value).abs() - bound
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0, (what, worst, value.abs().max().item(), bound.max().item())


def inputs(P, V, D, dtype, seed, scale=1.0, ignored=0.0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g) / D ** 0.5
    labels = torch.randint(0, V, (P,), generator=g)
    x = torch.randn(P, D, generator=g) + w[labels]
    labels[torch.rand(P, generator=g) < ignored] = IGN
    return x.to(dtype).cuda(), w.to(dtype).cuda(), labels.cuda()


def check(x, w, labels, scale=1.0, reduction="mean", lse_weight=0.0, ignore=IGN, want=("x", "w"), dtype=None, n3=None):
    """One call with its gradients, every output against the reference.  A random row gradient for "none"."""
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    P = x.shape[0]
    g = torch.Generator().manual_seed(P + w.shape[0])
    per_row = torch.randn(P, generator=g).cuda()
    per_lse = (torch.randn(P, generator=g) * lse_weight).cuda()
    n = max(1, int((labels != ignore).sum()))
    up = {"none": per_row.double(), "sum": torch.full((P,), 0.7, dtype=torch.float64, device="cuda"),
          "mean": torch.full((P,), 0.7 / n, dtype=torch.float64, device="cuda")}[reduction]
    ref = reference(x.detach(), w.detach(), labels.long(), scale, up, per_lse.double(), ignore, dtype, n3)
    xr, wr = x.detach().requires_grad_("x" in want), w.detach().requires_grad_("w" in want)
    loss, lse = vocabulary_cross_entropy(xr, wr, labels, scale, ignore, reduction, return_lse=True)
    assert loss.dtype == lse.dtype == torch.float32
    value, bound = ref["loss"]
    if reduction == "none":
        close(loss, ref["loss"], "loss")
    else:
        k = 1.0 if reduction == "sum" else 1.0 / n
        close(loss, (value.sum() * k, bound.sum() * k + 2 * U * value.sum().abs() * k), "loss")
    close(lse, ref["lse"], "lse")
    total = (loss * per_row).sum() if reduction == "none" else loss * 0.7
    if lse_weight:
        total = total + (lse * per_lse).sum()
    leaves = [t for t, name in ((xr, "x"), (wr, "w")) if name in want]
    grads = dict(zip([name for name in ("x", "w") if name in want], torch.autograd.grad(total, leaves)))
    for name, got in grads.items():
        assert got.dtype == x.dtype
        close(got, ref["d" + name], "d" + name)
    return loss, lse, grads


# ---- without a GPU ----------------------------------------------------------------------------------------------------
def test_entry_points_validate_without_a_gpu():
    lib = _lib.load()
    assert lib.pr_vocab_ce_kept_bytes(0, 4, 8, 16) > 0 and lib.pr_vocab_ce_fwd_scratch_bytes(2, 4, 8, 16) > 0
    for bad in ((3, 4, 8, 16), (-1, 4, 8, 16), (0, -1, 8, 16), (0, 4, 0, 16), (0, 4, 8, 0), (0, 1 << 31, 8, 16),
                (0, 4, 1 << 31, 16), (0, 1 << 29, 8, 1 << 19)):
        assert lib.pr_vocab_ce_kept_bytes(*bad) == 0
        assert lib.pr_vocab_ce_fwd_scratch_bytes(*bad) == 0
        assert lib.pr_vocab_ce_bwd_scratch_bytes(*bad, 1, 1) == 0
    assert lib.pr_vocab_ce_bwd_scratch_bytes(0, 4, 8, 16, 0, 0) == 0
    # a piece of the vocabulary, not the logits: 64 K rows and 256 K words in less than 2 GiB beside the packed tables
    P, V, D = 65536, 262144, 64
    logits = P * V * 2
    assert lib.pr_vocab_ce_bwd_scratch_bytes(2, P, V, D, 1, 1) < logits / 16
    assert lib.pr_vocab_ce_fwd_scratch_bytes(2, P, V, D) < logits / 16
    buf = ctypes.create_string_buffer(4096)
    ok = ctypes.c_void_p((ctypes.addressof(buf) + 255) & ~255)
    odd = ctypes.c_void_p(ok.value + 1)

    def fwd(dtype=0, P=4, V=8, D=16, x=ok, ld=(16, 1), w=ok, labels=ok, scale=1.0, kept=ok, kb=1 << 30, scratch=ok, sb=1 << 30,
            row=ok):
        return lib.pr_vocab_ce_fwd(dtype, P, V, D, x, *ld, w, *ld, labels, -100, scale, 0, kept, kb, scratch, sb, row, None,
                                   None, None)      # row None: neither the rows' losses nor their sum are wanted

    for kw in (dict(dtype=3), dict(P=0), dict(V=0), dict(D=0), dict(x=None), dict(w=None), dict(labels=None), dict(x=odd),
               dict(labels=odd), dict(ld=(-1, 1)), dict(scale=math.nan), dict(scale=math.inf), dict(kept=None, P=0),
               dict(scratch=None), dict(row=None), dict(kept=odd), dict(scratch=odd),
               dict(kept=None, P=lib.pr_vocab_ce_score_rows() + 1), dict(kept=None, scratch=None)):
        assert fwd(**kw) == -1, kw
    assert fwd(kept=None, sb=16) == -3
    assert fwd(kb=16) == -3 and fwd(sb=16) == -3

    def bwd(dx=ok, dw=ok, kept=ok, kb=1 << 30, scratch=ok, sb=1 << 30, P=4):
        return lib.pr_vocab_ce_bwd(0, P, 8, 16, None, 0, 0, ok, -100, 1.0, 0, 0, kept, kb, ok, None, scratch, sb, dx, dw, None)

    assert bwd(dx=None, dw=None) == 0
    for kw in (dict(dx=odd), dict(dw=odd), dict(kept=None), dict(scratch=None), dict(scratch=odd), dict(P=0)):
        assert bwd(**kw) == -1, kw
    assert bwd(kb=16) == -3 and bwd(sb=16) == -3
    # few rows and a large vocabulary: the features' gradient reads the vocabulary again
    assert lib.pr_vocab_ce_keeps_vocabulary(4, 8, 16) == 1 and lib.pr_vocab_ce_keeps_vocabulary(4, 1 << 17, 16) == 0
    for w, ld in ((None, (16, 1)), (odd, (16, 1)), (ok, (-1, 1))):
        assert lib.pr_vocab_ce_bwd(0, 4, 1 << 17, 16, w, *ld, ok, -100, 1.0, 0, 0, ok, 1 << 30, ok, None, ok, 1 << 30, ok, ok,
                                   None) == -1
    assert lib.pr_vocab_ce_bwd(0, 4, 1 << 17, 16, ok, 16, 1, ok, -100, 1.0, 0, 0, ok, 16, ok, None, ok, 1 << 30, ok, ok, None) == -3


def test_refusals():
    from pogs_amd.vocabulary import vocabulary_cross_entropy as f

    x, w, y = torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="HIP device"):
        f(x, w, y)
    for args, error, match in (
            ((x, torch.zeros(5, 3), y), ValueError, "dims"), ((x, torch.zeros(4), y), ValueError, "words, dims"),
            ((x, torch.zeros(0, 4), y), ValueError, "not empty"), ((x, w, y[:2]), ValueError, "labels"),
            ((x, w, y.float()), TypeError, "int64"), ((x, w.half(), y), TypeError, "both"),
            ((x.double(), w.double(), y), TypeError, "both")):
        with pytest.raises(error, match=match):
            f(*args)
    for kw, error, match in ((dict(scale=math.nan), ValueError, "finite"), (dict(scale=math.inf), ValueError, "finite"),
                             (dict(scale=torch.ones(())), TypeError, "plain number"),
                             (dict(reduction="max"), ValueError, "reduction")):
        with pytest.raises(error, match=match):
            f(x, w, y, **kw)


def test_scale_whose_logits_cannot_be_formed_is_refused():
    from pogs_amd.vocabulary import vocabulary_cross_entropy as f

    x, w, y = torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
    at, n = ctypes.c_void_p(1 << 20), 1 << 30
    lib = _lib.load()
    for scale in (1.1e38, -3e38):      # times log2(e), 3e38 is infinite
        with pytest.raises(ValueError, match="finite"):
            f(x, w, y, scale=scale)
        assert lib.pr_vocab_ce_fwd(0, 3, 5, 4, at, 4, 1, at, 4, 1, at, -100, scale, 0, at, n, at, n, at, None, None, None) == -1
        assert lib.pr_vocab_ce_bwd(0, 3, 5, 4, at, 4, 1, at, -100, scale, 0, 1, at, n, at, None, at, n, at, at, None) == -1
    with pytest.raises(RuntimeError, match="HIP device"):
        f(x, w, y, scale=1e38)


# ---- on the GPU -------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 2, 3), (5, 7, 9), (2, 300, 33), (33, 256, 32), (128, 257, 64), (129, 511, 65), (300, 1000, 128),
          (64, 5001, 96), (257, 513, 520), (1000, 77, 100), (31, 2048, 200)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("P,V,D", SHAPES)
def test_shapes_and_types(P, V, D, dtype):
    x, w, y = inputs(P, V, D, dtype, seed=P + V + D, ignored=0.2 if P > 4 else 0.0)
    check(x, w, y, reduction="mean")
    check(x, w, y, scale=3.0, reduction="none", lse_weight=1.0)
    check(x, w, y, scale=-2.5, reduction="sum", lse_weight=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_one_gradient_at_a_time_and_only_the_log_sum(dtype):
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, y = inputs(150, 700, 72, dtype, seed=1, ignored=0.3)
    _, _, both = check(x, w, y, reduction="none", lse_weight=1.0)
    for want in (("x",), ("w",)):
        _, _, one = check(x, w, y, reduction="none", lse_weight=1.0, want=want)
        assert torch.equal(one[want[0]], both[want[0]])
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    _, lse = vocabulary_cross_entropy(xr, wr, y, return_lse=True)
    gx, gw = torch.autograd.grad(lse.sum(), (xr, wr))
    ref = reference(x, w, y, 1.0, torch.zeros(150, device="cuda", dtype=torch.float64),
                    torch.ones(150, device="cuda", dtype=torch.float64))
    close(gx, ref["dx"], "dx")
    close(gw, ref["dw"], "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["f32", "f16"])
def test_strides_and_layouts(dtype):
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, y = inputs(90, 400, 70, dtype, seed=5, ignored=0.1)
    loss, lse, grads = check(x, w, y)
    wide = torch.full((90, 150), float("nan"), dtype=dtype, device="cuda")
    for xs, ws in ((x.t().contiguous().t(), w.t().contiguous().t()),
                   (wide[:, 3:143:2].copy_(x), torch.stack([w, w * 2], 2)[:, :, 0]),
                   (x, torch.cat([w, w], 1)[:, :70])):
        l2, s2, g2 = check(xs, ws, y.int())
        assert torch.equal(l2, loss) and torch.equal(s2, lse)
        assert all(torch.equal(g2[k], grads[k]) for k in grads)
    # leading dimensions, and rows shared by expansion: the gradient of the shared row is the sum
    xr = x.clone().requires_grad_(True)
    out = vocabulary_cross_entropy(xr.view(9, 10, 70), w, y.view(9, 10), reduction="none")
    assert out.shape == (9, 10)
    assert torch.equal(out.view(-1), vocabulary_cross_entropy(x, w, y, reduction="none"))
    assert torch.autograd.grad(out.sum(), xr)[0].shape == (90, 70)
    one = x[3:4].clone().requires_grad_(True)
    labels = torch.arange(40, device="cuda")
    total = vocabulary_cross_entropy(one.expand(40, 70), w, labels, reduction="sum")
    ref = reference(one.detach().expand(40, 70), w, labels, 1.0, torch.ones(40, device="cuda", dtype=torch.float64),
                    torch.zeros(40, device="cuda", dtype=torch.float64))
    value, bound = ref["dx"]
    got = torch.autograd.grad(total, one)[0]
    # torch adds the 40 rows' gradients in float32 or wider and rounds once to the type
    close(got, (value.sum(0, keepdim=True), bound.sum(0, keepdim=True) + (40 * U + HALF[dtype]) * value.abs().sum(0)), "shared")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_ignored_rows_hold_anything(dtype):
    """NaN and infinities in rows without a label change nothing; a table whose ignore index is one of its words."""
    x, w, y = inputs(140, 333, 48, dtype, seed=11)
    for ignore in (IGN, 7):
        lab = y.clone()
        lab[::3] = ignore
        loss, lse, grads = check(x, w, lab, ignore=ignore)
        bad = x.clone()
        rows = torch.nonzero(lab == ignore)[:, 0]
        bad[rows[0]], bad[rows[1]], bad[rows[2], 5] = math.nan, math.inf, -math.inf
        bad[rows[3:6]] = torch.finfo(dtype).max
        l2, s2, g2 = check(bad, w, lab, ignore=ignore)
        assert torch.equal(loss, l2) and torch.equal(lse, s2)
        assert torch.equal(grads["x"], g2["x"]) and torch.equal(grads["w"], g2["w"])
        assert float(g2["x"][rows].abs().max()) == 0.0 and float(s2[rows].detach().abs().max()) == 0.0


@pytest.mark.gpu
def test_no_row_with_a_label_and_no_rows():
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, _ = inputs(20, 50, 16, torch.float32, seed=2)
    y = torch.full((20,), IGN, device="cuda")
    for P in (20, 0):
        for reduction, value in (("mean", math.nan), ("sum", 0.0), ("none", 0.0)):
            xr, wr = x[:P].clone().requires_grad_(True), w.clone().requires_grad_(True)
            loss = vocabulary_cross_entropy(xr, wr, y[:P], reduction=reduction)
            if reduction == "none":
                assert loss.shape == (P,) and not loss.abs().sum().item()
            else:
                assert loss.shape == () and (math.isnan(loss.item()) if reduction == "mean" else loss.item() == value)
            gx, gw = torch.autograd.grad(loss.sum(), (xr, wr))
            assert gx.shape == (P, 16) and gw.shape == (50, 16)
            assert not gx.abs().sum().item() and not gw.abs().sum().item()


@pytest.mark.gpu
def test_labels_outside_the_vocabulary():
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, y = inputs(60, 100, 24, torch.float32, seed=3)
    plain = vocabulary_cross_entropy(x, w, y, reduction="none")        # few rows without gradients: kernels of their own
    good = vocabulary_cross_entropy(x.clone().requires_grad_(True), w, y, reduction="none")
    for bad in (100, -1, 1 << 40, -(1 << 40), 256, 127):
        lab = y.clone()
        lab[17] = bad
        loss = vocabulary_cross_entropy(x, w, lab, reduction="none")
        assert math.isnan(loss[17].item()) and torch.equal(loss[:17], plain[:17]) and torch.equal(loss[18:], plain[18:])
        xr = x.clone().requires_grad_(True)
        loss = vocabulary_cross_entropy(xr, w, lab, reduction="none")
        assert math.isnan(loss[17].item())
        rest = torch.arange(60, device="cuda") != 17
        assert torch.equal(loss[rest], good[rest])
        g = torch.autograd.grad(loss.sum(), xr)[0]
        assert torch.isnan(g[17]).all() and torch.isfinite(g[rest]).all()
        assert math.isnan(vocabulary_cross_entropy(x, w, lab).item())


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_with_their_rows():
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        x, w, y = inputs(70, 90, 40, dtype, seed=6)
        good = vocabulary_cross_entropy(x, w, y, reduction="none")
        x[5, 3], x[33, 0] = math.nan, math.inf
        loss = vocabulary_cross_entropy(x, w, y, reduction="none")
        rest = torch.ones(70, dtype=torch.bool, device="cuda")
        rest[5] = rest[33] = False
        assert torch.isnan(loss[~rest]).all() and torch.equal(loss[rest], good[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("exp_x,exp_w", [(90, -90), (-90, 90), (-60, 0), (0, 60), (-100, -100)])
def test_magnitudes(exp_x, exp_w):
    """Powers of two in features and vocabulary: the same bits where their product with the scale is the same, with and
    without gradients to come."""
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, y = inputs(40, 300, 64, torch.float32, seed=8)
    total = exp_x + exp_w
    for grads in (False, True):
        a, b = x.clone().requires_grad_(grads), w.clone().requires_grad_(grads)
        xs, ws = (x * 2.0 ** exp_x).requires_grad_(grads), (w * 2.0 ** exp_w).requires_grad_(grads)
        base = vocabulary_cross_entropy(a, b, y, reduction="none", return_lse=True)
        if total == -200:      # logits vanish: the loss is the logarithm of the number of words
            loss, _ = vocabulary_cross_entropy(xs, ws, y, reduction="none", return_lse=True)
            assert ((loss - math.log(300)).abs() <= 16 * U * math.log(300)).all()
            continue
        loss, lse = vocabulary_cross_entropy(xs, ws, y, scale=2.0 ** -total, reduction="none", return_lse=True)
        assert torch.equal(loss, base[0]) and torch.equal(lse, base[1])
        if grads:
            for got, want, e in zip(torch.autograd.grad(loss.sum(), (xs, ws)), torch.autograd.grad(base[0].sum(), (a, b)),
                                    (exp_x, exp_w)):
                assert torch.equal(got * 2.0 ** e, want)


@pytest.mark.gpu
def test_half_precision_below_its_normal_range():
    """float16 features of a few steps of 2^-24: the matrix cores take them as they are.  (The features' gradient, 2^20
    times a mean of the vocabulary, is beyond float16.)"""
    g = torch.Generator().manual_seed(12)
    w = torch.randn(200, 64, generator=g).half().cuda()
    x = (torch.randint(-40, 41, (70, 64), generator=g).double() * 2.0 ** -24).half().cuda()
    y = torch.randint(0, 200, (70,), generator=g).cuda()
    check(x, w, y, scale=2.0 ** 20, reduction="none", want=("w",))
    z = torch.zeros(64, device="cuda", dtype=torch.float64)
    from pogs_amd.vocabulary import vocabulary_cross_entropy
    close(vocabulary_cross_entropy(x[:64], w, y[:64], 2.0 ** 20, reduction="none"),
          reference(x[:64], w, y[:64], 2.0 ** 20, z, z)["loss"], "few rows")


@pytest.mark.gpu
def test_large_logits_and_mixed_row_sizes():
    x, w, y = inputs(64, 500, 64, torch.float32, seed=13)
    check(x, w, y, scale=2000.0, reduction="none", lse_weight=0.5)     # logits of thousands, probabilities 0 and 1
    x = x * torch.logspace(-6, 3, 64, device="cuda")[:, None]
    check(x, w, y, reduction="none")
    check(x, w, y, reduction="sum")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("P,V,D", [(1, 1, 1), (1, 33, 64), (1, 40_000, 512), (5, 31, 7), (31, 257, 65), (32, 1000, 130),
                                   (33, 999, 256), (63, 64, 1030), (64, 5000, 100), (65, 300, 72), (24, 33_000, 96)])
def test_scoring_without_gradients(P, V, D, dtype):
    """Few rows and no gradient to come: the vocabulary is read as it is.  float32 values are cut into three pieces of
    eight bits by truncation; the products left out are below 2 * 2^-7 * 2^-15 + 2^-30 of their product (inside rho), and
    six passes are added (n3)."""
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, y = inputs(P, V, D, dtype, seed=P + V, ignored=0.2 if P > 4 else 0.0)
    z = torch.zeros(P, device="cuda", dtype=torch.float64)
    wide = torch.full((P, D + 24), float("nan"), dtype=dtype, device="cuda")
    for scale, layout in ((1.0, 0), (-7.0, 1), (30.0, 2)):
        xs, ws = x, w
        if layout == 1:
            xs, ws = wide[:, 8:D + 8].copy_(x), w.t().contiguous().t()
        elif layout == 2:
            xs, ws = wide[:, 3:D + 3].copy_(x), torch.cat([w, w], 1)[:, :D]
        ref = reference(x, w, y, scale, z, z, n3=6 if dtype == torch.float32 else 1)
        with torch.no_grad():
            loss, lse = vocabulary_cross_entropy(xs, ws.requires_grad_(layout == 0), y, scale, reduction="none", return_lse=True)
            total = vocabulary_cross_entropy(xs, ws, y, scale, reduction="sum")
        w.requires_grad_(False)
        close(loss, ref["loss"], "loss")
        close(lse, ref["lse"], "lse")
        close(total, (ref["loss"][0].sum(), ref["loss"][1].sum() + 2 * U * ref["loss"][0].sum().abs()), "sum")
        again = vocabulary_cross_entropy(xs, ws, y, scale, reduction="none")
        assert torch.equal(again, loss)


FEW_SHAPES = [(1, 40_000, 64), (5, 33_001, 65), (32, 16_384, 128), (33, 2049, 1030), (64, 9000, 520), (65, 4200, 500),
              (100, 131_073, 16), (127, 300_001, 7), (128, 21_001, 100), (40, 33_000, 130), (64, 40_001, 33), (96, 32_768, 200), (17, 3, 700_001), (2, 3, 1_040_000)]
FEW_PASSES = {torch.float32: 6, torch.float16: 1, torch.bfloat16: 2}     # products added for one of operands


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("P,V,D", FEW_SHAPES)
def test_few_rows_and_a_large_vocabulary(P, V, D, dtype):
    """The vocabulary is not packed: float32 products as in scoring (left out: less than rho), a bfloat16 vocabulary meets
    G in two pieces (2^-14 of an entry, inside its rounding to float16)."""
    assert not _lib.load().pr_vocab_ce_keeps_vocabulary(P, V, D)
    x, w, y = inputs(P, V, D, dtype, seed=P + V + D, ignored=0.2 if P > 4 else 0.0)
    n3 = FEW_PASSES[dtype]
    check(x, w, y, scale=3.0, reduction="none", lse_weight=1.0, n3=n3)
    check(x, w, y, scale=-2.5, n3=n3)
    check(x, w, y, reduction="sum", want=("x",), n3=n3)
    check(x, w, y, want=("w",), n3=n3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
def test_few_rows_layouts(dtype):
    P, V, D = 40, 30_000, 75
    x, w, y = inputs(P, V, D, dtype, seed=3, ignored=0.2)
    want = check(x, w, y, scale=2.0, n3=FEW_PASSES[dtype])
    wide = torch.full((V, D + 24), float("nan"), dtype=dtype, device="cuda")
    for xs, ws in ((x, wide[:, 3:D + 3].copy_(w)), (x.t().contiguous().t(), w), (x, w.t().contiguous().t()),
                   (torch.cat([x, x])[::2].copy_(x), torch.cat([w, w], 1).view(V, 2, D)[:, 0])):
        got = check(xs, ws, y, scale=2.0, n3=FEW_PASSES[dtype])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert all(torch.equal(got[2][k], want[2][k]) for k in "xw")
    one = w[:1].expand(V, D)                    # every word the same: probabilities 1 / V, a broadcast vocabulary's gradient
    check(x, one, y, scale=2.0, n3=FEW_PASSES[dtype])
    check(x[:1].expand(P, D), w, y, scale=2.0, n3=FEW_PASSES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("P,V", [(20, 30_000), (20, 40_000), (50, 30_000), (50, 40_000), (70, 30_000), (128, 40_000)])
def test_few_rows_what_is_masked_or_not_finite(P, V, dtype):
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, y = inputs(P, V, 72, dtype, seed=5)
    row = torch.arange(P, device="cuda")

    def step(x, y, ignore=IGN):
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss, lse = vocabulary_cross_entropy(a, b, y, 2.0, ignore, "none", return_lse=True)
        with torch.no_grad():
            again = vocabulary_cross_entropy(a, b, y, 2.0, ignore, "none")
        assert ((again == loss) | torch.isnan(loss)).all()
        return (loss.detach(), lse.detach()) + torch.autograd.grad(loss.sum() + lse[10:].sum(), (a, b))

    x2, y2 = x.clone(), y.clone()
    x2[:3], x2[3:6], x2[6:9] = math.nan, math.inf, torch.finfo(dtype).min
    y2[:9] = 12                                 # ignored rows hold anything; the ignored label may be a word's
    y2[9:][y2[9:] == 12] = 13
    got, want = step(x2, y2, 12), step(x, torch.where(row < 9, IGN, y2))
    assert all(torch.equal(p, q) and torch.isfinite(p).all() for p, q in zip(got, want))
    assert (got[0][:9] == 0).all() and (got[1][:9] == 0).all() and (got[2][:9] == 0).all()
    none = step(x, torch.full_like(y, IGN))     # nothing left
    assert all((t == 0).all() for t in none)
    for bad in (V, -1, 1 << 40):                # a label that no word has
        y3 = y.clone()
        y3[11] = bad
        got = step(x, y3)
        assert torch.isnan(got[0][11]) and torch.isfinite(got[0][row != 11]).all() and torch.isfinite(got[1]).all()
        assert torch.isnan(got[2][11]).all() and torch.isfinite(got[2][row != 11]).all() and torch.isnan(got[3]).all()
    x4 = x.clone()
    x4[P - 3, 1] = math.nan                     # a row that is not finite
    got, want, rest = step(x4, y), step(x, y), row != P - 3
    assert torch.isnan(got[0][P - 3]) and torch.equal(got[0][rest], want[0][rest]) and torch.equal(got[2][rest], want[2][rest])


@pytest.mark.gpu
@pytest.mark.parametrize("P,V", [(40, 20_000), (20, 40_000), (100, 40_000)])
@pytest.mark.parametrize("exp_x,exp_w", [(90, -90), (-90, 90), (-60, 0), (0, 60), (-50, -50)])
def test_few_rows_magnitudes(exp_x, exp_w, P, V):
    """Nothing is scaled, and a power of two changes no bit of a piece or a product: the same bits as at 1."""
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, y = inputs(P, V, 32, torch.float32, seed=8)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    xs, ws = (x * 2.0 ** exp_x).requires_grad_(True), (w * 2.0 ** exp_w).requires_grad_(True)
    base = vocabulary_cross_entropy(a, b, y, reduction="none", return_lse=True)
    loss = vocabulary_cross_entropy(xs, ws, y, scale=2.0 ** -(exp_x + exp_w), reduction="none", return_lse=True)
    assert torch.equal(loss[0], base[0]) and torch.equal(loss[1], base[1])
    want = torch.autograd.grad(base[0].sum(), (a, b))
    for got, ref, e in zip(torch.autograd.grad(loss[0].sum(), (xs, ws)), want, (exp_x, exp_w)):
        assert torch.equal(got * 2.0 ** e, ref)


@pytest.mark.gpu
def test_few_rows_in_a_graph_and_a_vocabulary_that_changes():
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, y = inputs(48, 40_000, 60, torch.float32, seed=15, ignored=0.1)
    x.requires_grad_(True), w.requires_grad_(True)

    def step():
        loss = vocabulary_cross_entropy(x, w, y, 3.0)
        return (loss.detach(),) + torch.autograd.grad(loss, (x, w))

    eager = step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = step()
    for k in range(4):
        with torch.no_grad():
            x.mul_(0.5)
        want = step()
        for t in res:
            t.zero_()
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(res, want))
    assert not torch.equal(want[0], eager[0])
    loss = vocabulary_cross_entropy(x, w, y, 3.0)
    with torch.no_grad():
        w.mul_(2.0)                             # the backward pass would read it: refused
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, (x, w))


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences of the float64 loss, at steps small enough for 1e-5 of the gradient's scale."""
    x, w, y = inputs(6, 40, 10, torch.float32, seed=21, ignored=0.2)
    _, _, grads = check(x, w, y, scale=4.0)
    x64, w64 = x.double(), w.double()

    def loss(a, b):
        return 0.7 * torch.nn.functional.cross_entropy(4.0 * a @ b.t(), y)      # check() takes 0.7 of the loss

    for which, t in (("x", x64), ("w", w64)):
        diff = torch.zeros_like(t)
        for i in range(t.numel()):
            e = torch.zeros_like(t).view(-1)
            e[i] = 1e-4
            e = e.view_as(t)
            if which == "x":
                diff.view(-1)[i] = (loss(x64 + e, w64) - loss(x64 - e, w64)) / 2e-4
            else:
                diff.view(-1)[i] = (loss(x64, w64 + e) - loss(x64, w64 - e)) / 2e-4
        # third derivatives of the loss: at most scale^3 |w|^3 (about 4^3 * 8): h^2 / 6 of them is below 1e-6
        assert ((grads[which].double() - diff).abs() <= 1e-6 + 1e-5 * diff.abs().max()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_a_vocabulary_in_several_pieces(dtype):
    P, V, D = (4096, 40_001, 40) if dtype == torch.float32 else (8192, 40_001, 40)
    lib = _lib.load()
    whole = P * ((V + 255) // 256 * 256) * 2 * 2 * NP[dtype]
    assert lib.pr_vocab_ce_bwd_scratch_bytes({torch.float32: 0, torch.bfloat16: 2}[dtype], P, V, D, 1, 1) < whole
    x, w, y = inputs(P, V, D, dtype, seed=17, ignored=0.1)
    check(x, w, y, scale=2.0)


@pytest.mark.gpu
def test_features_beyond_32_bit_offsets():
    P, V, D = (1 << 21) + 5, 260, 1030
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    g = torch.Generator(device="cuda").manual_seed(0)
    w = (torch.randn(V, D, generator=g, device="cuda") / 32).to(torch.bfloat16)
    x = torch.empty(P, D, dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 1 << 31
    x.normal_(generator=g)
    y = torch.randint(0, V, (P,), generator=g, device="cuda")
    xr = x.requires_grad_(True)
    loss = vocabulary_cross_entropy(xr, w, y, reduction="none")
    gx = torch.autograd.grad(loss.sum(), xr)[0]
    rows = torch.tensor([0, 1, 12_345, P // 2, P - 130, P - 129, P - 2, P - 1], device="cuda")
    ones = torch.ones(len(rows), device="cuda", dtype=torch.float64)
    ref = reference(x.detach()[rows], w, y[rows], 1.0, ones, 0 * ones)
    close(loss[rows], ref["loss"], "loss")
    close(gx[rows], ref["dx"], "dx")


@pytest.mark.gpu
def test_vocabulary_beyond_32_bit_offsets():
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    P, V, D = 5, (1 << 21) + 77, 1030
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.empty(V, D, dtype=torch.bfloat16, device="cuda")
    assert w.numel() > 1 << 31
    w.normal_(generator=g).mul_(0.125)
    x = torch.randn(P, D, generator=g, device="cuda").to(torch.bfloat16) * 0.25
    y = torch.tensor([0, V - 1, V - 78, 1 << 20, IGN], device="cuda")
    z = torch.cat([x.double() @ w[lo:lo + (1 << 18)].double().t() for lo in range(0, V, 1 << 18)], 1)
    lse = torch.logsumexp(z, 1)
    want = lse[:4] - z[torch.arange(4), y[:4]]
    wr = w.requires_grad_(True)
    loss = vocabulary_cross_entropy(x, wr, y, reduction="none")
    # |x| |w| of a row is about 0.25 * 0.125 * 1030 * 0.64: the logits' error is below 1e-4 by the bound above
    assert ((loss[:4].double() - want).abs() <= 1e-3).all() and loss[4].item() == 0.0
    with torch.no_grad():
        few = vocabulary_cross_entropy(x, w, y, reduction="none")
    assert ((few[:4].double() - want).abs() <= 1e-3).all()
    dw = torch.autograd.grad(loss.sum(), wr)[0]
    for v in (0, 1, V // 2, V - 78, V - 1):
        p = (z[:4, v] - lse[:4]).exp() - (y[:4] == v).double()
        ref = p @ x[:4].double()
        mag = p.abs() @ x[:4].double().abs()
        # logits 1e-3, G 2^-11, bf16 2^-8
        assert ((dw[v].double() - ref).abs() <= mag * (2e-3 + 2.0 ** -11) + ref.abs() * 2.0 ** -8 + 2.0 ** -40).all(), v


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("P,V,D", [(1, 1, 1), (3, 257, 31), (65, 700, 33), (257, 1300, 130), (600, 90, 96), (513, 5000, 520),
                                   (1, 40_000, 64), (33, 2049, 1030), (100, 33_001, 65)])
def test_nothing_is_written_outside_the_buffers(P, V, D, dtype):
    """Every buffer of the C entry points at its exact size between guard bytes."""
    lib, t = _lib.load(), {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    x, w, y = inputs(P, V, D, dtype, seed=3)
    guarded = []

    def buffer(nbytes):
        b = torch.full((nbytes + 8192,), 0x5A, dtype=torch.uint8, device="cuda")
        guarded.append((b, nbytes))
        return ctypes.c_void_p(b.data_ptr() + 4096)

    e = x.element_size()
    nk, nf = lib.pr_vocab_ce_kept_bytes(t, P, V, D), lib.pr_vocab_ce_fwd_scratch_bytes(t, P, V, D)
    st = torch.cuda.current_stream().cuda_stream

    def fwd(kept):
        return lib.pr_vocab_ce_fwd(t, P, V, D, x.data_ptr(), D, 1, w.data_ptr(), D, 1, y.data_ptr(), -100, 2.0, 1, kept, nk,
                                   buffer(nf), nf, buffer(4 * P), buffer(4 * P), buffer(4), st)

    kept = buffer(nk)
    assert fwd(kept) == 0
    if P <= lib.pr_vocab_ce_score_rows():
        assert fwd(None) == 0
    g = torch.ones(1, device="cuda")
    for dx, dw in ((1, 1), (1, 0), (0, 1)):
        nb = lib.pr_vocab_ce_bwd_scratch_bytes(t, P, V, D, dx, dw)
        assert lib.pr_vocab_ce_bwd(t, P, V, D, w.data_ptr(), D, 1, y.data_ptr(), -100, 2.0, 1, 0, kept, nk, g.data_ptr(), None, buffer(nb), nb,
                                   buffer(e * P * D) if dx else None, buffer(e * V * D) if dw else None, st) == 0
    torch.cuda.synchronize()
    for b, n in guarded:
        assert (b[:4096] == 0x5A).all() and (b[4096 + n:] == 0x5A).all()


@pytest.mark.gpu
def test_inputs_changed_after_the_forward_pass():
    """The backward pass has its own copy of features and vocabulary; changed labels are noticed."""
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, y = inputs(50, 120, 32, torch.float32, seed=9)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    want = torch.autograd.grad(vocabulary_cross_entropy(a, b, y), (a, b))
    a2, b2 = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = vocabulary_cross_entropy(a2, b2, y)
    with torch.no_grad():
        a2.zero_(), b2.mul_(3.0)
    got = torch.autograd.grad(loss, (a2, b2))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    loss = vocabulary_cross_entropy(a, b, y)
    y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, (a, b))


@pytest.mark.gpu
def test_equal_inputs_give_equal_bits():
    x, w, y = inputs(2000, 9000, 96, torch.float32, seed=30, ignored=0.1)
    first = check(x, w, y)
    for _ in range(3):
        again = check(x, w, y)
        assert torch.equal(first[0], again[0]) and all(torch.equal(first[2][k], again[2][k]) for k in "xw")


@pytest.mark.gpu
def test_graphs_and_streams():
    """Forward and backward captured into two graphs, replayed with eager work between; the same call on two streams at
    once; one forward pass with two backward passes on two streams."""
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x0, w0, y0 = inputs(300, 1000, 64, torch.float32, seed=40, ignored=0.1)
    x1, w1, y1 = inputs(200, 3000, 80, torch.bfloat16, seed=41)
    sets = [(x0.requires_grad_(True), w0.requires_grad_(True), y0), (x1.requires_grad_(True), w1.requires_grad_(True), y1)]

    def step(x, w, y):
        loss = vocabulary_cross_entropy(x, w, y, scale=3.0)
        return (loss.detach(),) + torch.autograd.grad(loss, (x, w))

    def same(a, b):
        return all(torch.equal(p, q) for p, q in zip(a, b))

    eager = [step(*s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    out = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            out.append([step(*s) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(same(o, e) for outs, e in zip(out, eager) for o in outs)

    loss = vocabulary_cross_entropy(*sets[0], scale=3.0)
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    twice = []
    for st, k in zip(streams, (1.0, 2.0 ** 20)):
        with torch.cuda.stream(st):
            twice.append(torch.autograd.grad(loss, sets[0][:2], grad_outputs=torch.tensor(k, device="cuda"), retain_graph=True))
    torch.cuda.synchronize()
    assert same(twice[0], eager[0][1:])
    assert all(torch.equal(a * 2.0 ** 20, b) for a, b in zip(*twice))

    # while the eager graph of the same leaves lives, capturing another one is refused
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step(*sets[0])
    del loss
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(*s)
        graphs.append((g, res))
    for i in range(3):
        fresh = [inputs(300, 1000, 64, torch.float32, seed=50 + i, ignored=0.2), inputs(200, 3000, 80, torch.bfloat16, seed=60 + i)]
        for s, f in zip(sets, fresh):
            for a, b in zip(s, f):
                a.detach().copy_(b)
        for g, _ in graphs:
            g.replay()
        torch.full((1 << 20,), 2.0, device="cuda").sum().item()
        for (g, res), s in zip(graphs, sets):
            assert same(res, step(*s))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["rows", "batch", "one row", "transposed"])
def test_capture_is_refused_while_a_graph_of_the_leaves_lives(layout):
    """Features that the call makes rows of itself are leaves all the same; nothing is captured past the refusal."""
    from pogs_amd.vocabulary import vocabulary_cross_entropy

    x, w, y = inputs(12, 50, 16, torch.float32, seed=44)
    x, y = {"rows": lambda: (x, y), "batch": lambda: (x.view(3, 4, 16), y.view(3, 4)), "one row": lambda: (x[0], y[0]),
            "transposed": lambda: (x.view(3, 4, 16).transpose(0, 1), y.view(3, 4).t())}[layout]()
    x = x.detach().requires_grad_(True)
    loss = vocabulary_cross_entropy(x, w, y)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            vocabulary_cross_entropy(x, w, y)
    eager, = torch.autograd.grad(loss, x)
    del loss
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured, = torch.autograd.grad(vocabulary_cross_entropy(x, w, y), x)
    for _ in range(3):
        captured.zero_()
        g.replay()
        assert torch.equal(captured, eager)


@pytest.mark.gpu
def test_training_step_of_heads_loss_clipping_and_adam():
    """The operators as they are used together: clip head -> vocabulary loss -> gradients -> step clipped to the head's
    own norm.  The head's products are split-bf16 (2^-16 each), four layers deep: 1e-4 of the loss.  A gradient through a
    ReLU is a step function of the pre-activation, and the head's error decides those within it of zero one way or the
    other; so the weights' gradient is held against the head's own backward pass (which is linear) of the loss's float64
    gradient at the head's output: u of each side, 1e-5 of the largest entry for four layers of 2^-16 on differences."""
    from oracle.heads_ref import dense_network_ref
    from pogs_amd.heads import FieldHeads
    from pogs_amd.optim import Optimizers

    heads = FieldHeads(clip_n_dims=64, device="cuda", seed=3)
    gen = torch.Generator().manual_seed(4)
    P, V = 400, 700
    feats, scale = torch.randn(P, 96, generator=gen), torch.rand(P, 1, generator=gen)
    words = torch.nn.functional.normalize(torch.randn(V, 64, generator=gen), dim=1)
    labels = torch.randint(0, V, (P,), generator=gen)
    labels[::7] = IGN
    params = heads.clip_net.params.detach().cpu().double()
    hidden, _ = dense_network_ref(torch.cat([feats.double(), scale.double()], 1), params, heads.clip_net.shapes, 97, 64)
    unit = hidden / hidden.norm(dim=1, keepdim=True)
    want = torch.nn.functional.cross_entropy(20.0 * unit @ words.double().t(), labels)

    clip = heads.get_clip_outputs_from_feature(feats.cuda(), scale.cuda())
    at = clip.detach().cpu().double().requires_grad_(True)
    torch.nn.functional.cross_entropy(20.0 * at @ words.double().t(), labels).backward()
    ref = torch.autograd.grad(clip, heads.clip_net.params, grad_outputs=at.grad.float().cuda())[0].cpu().double()
    norm = ref.norm().item()

    opt = Optimizers({"clip": {"lr": 1e-3, "max_norm": 0.25 * norm}}, {"clip": [heads.clip_net.params]})
    opt.zero_grad_all()
    loss = heads.get_vocabulary_loss_from_feature(feats.cuda(), scale.cuda(), words.cuda(), labels.cuda(), logit_scale=20.0)
    loss.backward()
    opt.optimizer_step_all()
    assert abs(loss.item() - want.item()) <= 1e-4 * abs(want.item())
    got = heads.clip_net.params.grad.cpu().double()
    assert (got - ref).abs().max().item() <= 1e-5 * ref.abs().max().item()
    assert abs(opt.grad_norms["clip"].item() - norm) <= 1e-5 * norm
    # the first moment of a first step is a tenth of the clipped gradient
    m = opt.state("clip")["exp_avg"].cpu().double()
    assert abs(m.norm().item() - 0.1 * 0.25 * norm) <= 1e-5 * norm
    assert (m * 40 - got).abs().max().item() <= 2e-5 * got.abs().max().item()
