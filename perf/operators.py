"""What is measured of the vocabulary loss and of gradient clipping, and their plain forms.

Four kinds of case, by ``case["op"]``:

``score``  cross entropy of feature rows over a large vocabulary of embeddings, forward only: every row's negative log
           probability of its label and its log partition sum.
``train``  the same loss averaged over the rows that are not ignored, with its gradients.
``clip``   global 2-norm of the gradients of many tensors, and their scaling to at most ``max_norm``, in place.
``step``   one Adam step of several parameter groups, each group's gradient clipped to its own norm.

``own`` false: elementary torch operations in 32 bits (64 where a sum is long).  ``own`` true: the calls a user of the
framework makes.
"""
import math

import torch

own = False

IGNORE = -100
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

# per-Gaussian widths of the trained tensors of a scene: means, colour, the other harmonics, opacity, scales,
# rotations, feature channels
SCENE = (3, 3, 45, 1, 3, 4, 64)
# the trained tensors next to a scene: the clip and the instance head's flat weights, the channel network's four matrices
HEADS = (256 * 112 + 2 * 256 * 256 + 512 * 256, 256 * 96 + 3 * 256 * 256 + 128 * 256, 4096, 4096, 4096, 4096)


def listed():
    return [
        # one pixel's clip feature against a table of phrases: a user's click, where latency counts
        dict(name="score_one", op="score", rows=1, words=32000, dim=512, dtype="f32", scale=100.0, ignored=0.0),
        # two dozen objects' mean features labelled over a large table kept in 16 bits
        dict(name="score_few_bf16", op="score", rows=24, words=131072, dim=1024, dtype="bf16", scale=1.0, ignored=0.0),
        # an evaluation image's worth of random pixels over a label set of odd size
        dict(name="score_image_f32", op="score", rows=4099, words=20011, dim=512, dtype="f32", scale=100.0, ignored=0.1),
        # instance prototypes: a small table that is learned with the features
        dict(name="train_small_f32", op="train", rows=257, words=1000, dim=128, dtype="f32", scale=10.0, ignored=0.05,
             to_words=True),
        # a training batch of pixels against a frozen table of phrase embeddings: gradient to the features alone
        dict(name="train_frozen_f32", op="train", rows=4096, words=10000, dim=512, dtype="f32", scale=100.0, ignored=0.1,
             to_words=False),
        # odd sizes in half precision, a third of the pixels without a label, both gradients
        dict(name="train_ragged_f16", op="train", rows=1999, words=50021, dim=768, dtype="f16", scale=1.0, ignored=0.33,
             to_words=True),
        # the largest table and batch, both gradients
        dict(name="train_large_bf16", op="train", rows=8192, words=131072, dim=1024, dtype="bf16", scale=1.0, ignored=0.0,
             to_words=True),
        # the heads and the channel network: six small tensors, where latency counts
        dict(name="clip_heads", op="clip", layout="heads", count=6, size=0, dtype="f32"),
        # many tensors of ragged sizes, in 32 and in 16 bits
        dict(name="clip_mixed", op="clip", layout="mixed", count=56, size=2_000_003, dtype="mixed"),
        # a scene of a million Gaussians
        dict(name="clip_scene", op="clip", layout="scene", count=len(SCENE), size=1_000_000, dtype="f32"),
        # the optimiser step of the heads and the channel network, each group clipped by itself
        dict(name="step_heads", op="step", layout="heads", count=6, size=0, dtype="f32"),
        # the optimiser step of a scene of a million Gaussians
        dict(name="step_scene", op="step", layout="scene", count=len(SCENE), size=1_000_000, dtype="f32"),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "score", "train", "train", "clip", "step"])
    if op in ("score", "train"):
        while True:
            case = dict(op=op, rows=_log_between(rng, 1, 8192), words=_log_between(rng, 100, 131072),
                        dim=_log_between(rng, 64, 1024), dtype=rng.choice(["f32", "bf16", "f16"]),
                        ignored=round(rng.uniform(0.0, 0.4), 3))
            if rng.random() < 0.5:      # widths of real networks are multiples of 64 as often as not
                case["dim"] = max(64, case["dim"] // 64 * 64)
            case["scale"] = round(rng.uniform(5.0, 100.0), 2) if case["dtype"] == "f32" else 1.0
            if op == "train":
                case["to_words"] = rng.random() < 0.6
            if case["rows"] * case["words"] * case["dim"] <= 2 ** 38:
                return case
    layout = rng.choice(["scene", "mixed"])
    if op == "step" or layout == "scene":
        return dict(op=op, layout="scene", count=len(SCENE), size=_log_between(rng, 1000, 1_000_000), dtype="f32")
    return dict(op=op, layout="mixed", count=rng.randint(2, 60), size=_log_between(rng, 100, 2_000_003), dtype="mixed")


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _sizes(case):
    """[(elements, dtype)] of a gradient case's tensors."""
    if case["layout"] == "heads":
        return [(n, torch.float32) for n in HEADS]
    if case["layout"] == "scene":
        return [(w * case["size"], torch.float32) for w in SCENE]
    out = []
    for i in range(case["count"]):     # from a handful of values up to `size`, evenly in the logarithm; odd mostly
        n = max(1, int(case["size"] ** ((i + 1) / case["count"])))
        out.append((n, (torch.float32, torch.bfloat16, torch.float32, torch.float16)[i % 4]))
    return out


def _tables(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    P, V, D = case["rows"], case["words"], case["dim"]
    words = torch.randn(V, D, generator=g, device="cuda")
    labels = torch.randint(0, V, (P,), generator=g, device="cuda")
    feats = torch.randn(P, D, generator=g, device="cuda")
    if case["dtype"] == "f32":         # rows of length one, features that lean towards their label's embedding
        words /= words.norm(dim=1, keepdim=True)
        feats = feats / feats.norm(dim=1, keepdim=True) + 0.12 * words[labels]
        feats /= feats.norm(dim=1, keepdim=True)
    else:                              # a network's last activations: logits of a few units
        words *= D ** -0.5
        feats = feats + D ** 0.5 * words[labels] * 0.2
    drop = torch.rand(P, generator=g, device="cuda") < case["ignored"]
    drop[:1] = False
    labels[drop] = IGNORE
    dt = DTYPES[case["dtype"]]
    return feats.to(dt), words.to(dt), labels


def prepare(case, seed):
    if case["op"] in ("score", "train"):
        feats, words, labels = _tables(case, seed)
        s = dict(case=case, feats=feats, words=words, labels=labels)
        if case["op"] == "train":
            feats.requires_grad_(True)
            words.requires_grad_(case["to_words"])
        if own:
            from pogs_amd.vocabulary import vocabulary_cross_entropy
            s["call"] = vocabulary_cross_entropy
        return s
    g = torch.Generator(device="cuda").manual_seed(seed)
    params, total = [], 0
    for i, (n, dt) in enumerate(_sizes(case)):
        p = torch.randn(n, generator=g, device="cuda").mul_(0.1).to(dt).requires_grad_(True)
        p.grad = torch.randn(n, generator=g, device="cuda").mul_(0.01 * (1 + i % 3)).to(dt)
        total += n * (0.01 * (1 + i % 3)) ** 2
        params.append(p)
    # half of what the norm is expected to be: clipping is active
    s = dict(case=case, params=params, max_norm=0.5 * math.sqrt(total), names=["group%d" % i for i in range(len(params))])
    if case["op"] == "clip":
        if own:
            from pogs_amd.optim import clip_grad_norm_
            s["call"] = clip_grad_norm_
        return s
    # an optimiser that has taken a hundred steps
    s["steps"] = 100
    s["lr"] = [1e-3 * (1 + i % 5) for i in range(len(params))]
    s["max"] = [0.5 * 0.01 * (1 + i % 3) * math.sqrt(p.numel()) for i, p in enumerate(params)]
    s["exp_avg"] = [torch.randn(p.numel(), generator=g, device="cuda").mul_(0.005) for p in params]
    s["exp_avg_sq"] = [torch.rand(p.numel(), generator=g, device="cuda").mul_(2e-4).add_(1e-6) for p in params]
    if own:
        from pogs_amd.optim import Optimizers
        cfg = {n: {"lr": lr, "eps": 1e-15, "max_norm": m} for n, lr, m in zip(s["names"], s["lr"], s["max"])}
        s["opt"] = Optimizers(cfg, {n: [p] for n, p in zip(s["names"], params)})
        s["opt"].load_optimizers({n: {"state": {0: {"step": 100, "exp_avg": m, "exp_avg_sq": v}}}
                                  for n, m, v in zip(s["names"], s["exp_avg"], s["exp_avg_sq"])})
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def _plain_loss(s):
    case = s["case"]
    x, w, labels = s["feats"].detach().float(), s["words"].detach().float(), s["labels"]
    keep = labels != IGNORE
    at = labels.clamp(min=0)[:, None]
    z = (x @ w.t()).mul_(case["scale"])
    top = z.amax(dim=1, keepdim=True)
    lse = top + (z - top).exp().sum(dim=1, keepdim=True).log()
    loss = (lse - z.gather(1, at))[:, 0] * keep
    if case["op"] == "score":
        return {"loss": loss, "lse": lse[:, 0] * keep}
    n = keep.sum()
    p = z.sub_(lse).exp_()
    p.scatter_add_(1, at, -torch.ones_like(lse))
    p.mul_((keep * (case["scale"] / n))[:, None])
    out = {"loss": loss.sum() / n, "to_feats": (p @ w).to(s["feats"].dtype)}
    if case["to_words"]:
        out["to_words"] = (p.t() @ x).to(s["words"].dtype)
    return out


def _plain_norm(grads):
    return torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()


def _plain_clip(s):
    grads = [p.grad for p in s["params"]]
    norm = _plain_norm(grads)
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    [g.copy_(g.float() * coef) for g in grads]
    return {"norm": norm.float(), "grads": grads}


def _plain_adam(p, g, m, v, lr, max_norm, t):
    norm = _plain_norm([g])
    g = g * (max_norm / (norm + 1e-6)).clamp(max=1.0).float()
    m.lerp_(g, 0.1)
    v.mul_(0.999).addcmul_(g, g, value=0.001)
    p.sub_(m / (v.sqrt() / math.sqrt(1 - 0.999 ** t) + 1e-15) * (lr / (1 - 0.9 ** t)))
    return norm.float()


def run(state):
    s, op = state, state["case"]["op"]
    if op == "score":
        if not own:
            return _plain_loss(s)
        with torch.no_grad():
            loss, lse = s["call"](s["feats"], s["words"], s["labels"], scale=s["case"]["scale"], reduction="none",
                                  return_lse=True)
        return {"loss": loss, "lse": lse}
    if op == "train":
        if not own:
            return _plain_loss(s)
        loss = s["call"](s["feats"], s["words"], s["labels"], scale=s["case"]["scale"])
        wanted = [s["feats"]] + ([s["words"]] if s["case"]["to_words"] else [])
        grads = torch.autograd.grad(loss, wanted)
        out = {"loss": loss.detach(), "to_feats": grads[0]}
        if s["case"]["to_words"]:
            out["to_words"] = grads[1]
        return out
    if op == "clip":
        s["max_norm"] *= 0.999         # lowered a little each pass: clipping stays active on gradients once clipped
        if not own:
            return _plain_clip(s)
        norm = s["call"](s["params"], s["max_norm"])
        return {"norm": norm, "grads": [p.grad for p in s["params"]]}
    if not own:
        s["steps"] += 1
        with torch.no_grad():
            norms = [_plain_adam(p, p.grad, m, v, lr, mx, s["steps"]) for p, m, v, lr, mx in
                     zip(s["params"], s["exp_avg"], s["exp_avg_sq"], s["lr"], s["max"])]
        return {"norms": torch.stack(norms), "params": [p.detach() for p in s["params"]], "exp_avg": s["exp_avg"],
                "exp_avg_sq": s["exp_avg_sq"]}
    opt = s["opt"]
    opt.optimizer_step_all()
    st = [opt.state(n, 0) for n in s["names"]]
    return {"norms": torch.stack([opt.grad_norms[n] for n in s["names"]]), "params": [p.detach() for p in s["params"]],
            "exp_avg": [x["exp_avg"] for x in st], "exp_avg_sq": [x["exp_avg_sq"] for x in st]}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    if case["op"] in ("score", "train"):
        P, V, D, e = case["rows"], case["words"], case["dim"], BYTES[case["dtype"]]
        tables, product = (P + V) * D * e, 2.0 * P * V * D
        if case["op"] == "score":
            return {"bytes": tables + P * 16, "flops": product}
        grads = (P + (V if case["to_words"] else 0)) * D * e
        return {"bytes": tables + P * 8 + grads, "flops": product * (3 if case["to_words"] else 2)}
    sizes = _sizes(case)
    if case["op"] == "clip":           # read, and written scaled
        return {"bytes": sum(2 * n * dt.itemsize for n, dt in sizes), "flops": sum(3 * n for n, _ in sizes)}
    return {"bytes": sum(28 * n for n, _ in sizes), "flops": sum(15 * n for n, _ in sizes)}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("score", "train"):
        feats, words, labels = _tables(case, seed)
        x, w = feats.double(), words.double()
        P, V, D = case["rows"], case["words"], case["dim"]
        kept = torch.nonzero(labels != IGNORE)[:, 0]
        nll, lse = x.new_zeros(P), x.new_zeros(P)
        gx, gw = torch.zeros_like(x), torch.zeros_like(w) if case.get("to_words") else None
        rows = max(1, 2 ** 28 // V)
        for lo in range(0, len(kept), rows):
            r = kept[lo:lo + rows]
            z = case["scale"] * torch.mm(x[r], w.T)
            a = torch.logsumexp(z, dim=1)
            lse[r] = a
            nll[r] = a - z[torch.arange(len(r), device=z.device), labels[r]]
            if case["op"] == "train":
                q = torch.softmax(z, dim=1)
                q[torch.arange(len(r), device=z.device), labels[r]] -= 1.0
                q *= case["scale"] / len(kept)
                gx[r] = torch.mm(q, w)
                if gw is not None:
                    gw += torch.mm(q.T.contiguous(), x[r])
        if case["op"] == "score":
            return {"loss": nll, "lse": lse}
        out = {"loss": nll.sum() / len(kept), "to_feats": gx}
        if gw is not None:
            out["to_words"] = gw
        return out
    s = prepare(case, seed)
    grads = [p.grad.to(torch.float64) for p in s["params"]]
    if case["op"] == "clip":
        norm = math.sqrt(math.fsum(float((g * g).sum()) for g in grads))
        scale = min(1.0, 0.999 * s["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [g * scale for g in grads]}
    norms, ps, ms, vs = [], [], [], []
    first, second = 1 - 0.9 ** 101, 1 - 0.999 ** 101
    for p, g, m, v, lr, mx in zip(s["params"], grads, s["exp_avg"], s["exp_avg_sq"], s["lr"], s["max"]):
        norm = math.sqrt(float((g * g).sum()))
        g = g * min(1.0, mx / (norm + 1e-6))
        m, v = 0.9 * m.double() + 0.1 * g, 0.999 * v.double() + 0.001 * g * g
        ps.append(p.detach().double() - lr * (m / first) / ((v / second).sqrt() + 1e-15))
        ms.append(m)
        vs.append(v)
        norms.append(norm)
    return {"norms": torch.tensor(norms, dtype=torch.float64), "params": ps, "exp_avg": ms, "exp_avg_sq": vs}
