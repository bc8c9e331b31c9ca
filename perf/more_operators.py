"""Operators of training on one's own answers, and what is measured of them.

A classifier that is trained by rewards, on pseudo labels or towards sure
answers needs the log probabilities of given classes, the entropy of every
row and their gradients, and then clips its gradients:

  linear  layers.linear_log_probs: log probabilities of the given classes of
          softmax((hidden[rows] weight^T + bias) / T) (a negative index: none
          given, 0), every row's entropy, with top > 0 the largest logits'
          log probabilities and classes (ties: the lowest class), and the
          gradients of the log probabilities and the entropies.  The logits
          are not kept
  kept    layers.log_probs: the same of logits in memory
  clip    core.clip_grads: the norm over many gradients, and what is left of
          each where it is clipped, in f32
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one node answered from a vocabulary, as a served request is: its
        # answer's log probability, how sure it is, and eight alternatives
        dict(name="linear_answer_one_bf16", kind="linear", nodes=1, rows=1, width=2048, classes=32000, k=1, top=8,
             temperature=1.0, dtype="bf16", bias=False, grad=False, none=0.0),
        # a mini-batch step of the sampled configuration: 1,024 seeds, hidden
        # width 256, 172 classes, f16 under a loss scale
        dict(name="linear_batch_f16", kind="linear", nodes=1024, rows=1024, width=256, classes=172, k=1, top=0,
             temperature=1.0, dtype="f16", bias=True, grad=True, none=0.0),
        # sampled answers over a catalogue at hidden width 256, some rows
        # without one (their entropy still counts)
        dict(name="linear_catalogue_bf16", kind="linear", nodes=16384, rows=16384, width=256, classes=100003, k=1,
             top=0, temperature=1.0, dtype="bf16", bias=False, grad=True, none=0.1),
        # several candidates a row, the default precision, rows of a node
        # table, ragged sizes, an exploring temperature
        dict(name="linear_candidates_f32", kind="linear", nodes=4099, rows=3001, width=250, classes=10007, k=20,
             top=0, temperature=1.5, dtype="f32", bias=True, grad=True, none=0.05),
        # the largest: a vocabulary of 131,072 at width 4,096
        dict(name="linear_vocabulary_bf16", kind="linear", nodes=8192, rows=8192, width=4096, classes=131072, k=1,
             top=0, temperature=1.0, dtype="bf16", bias=False, grad=True, none=0.05),
        # scoring a batch's candidates with sixteen alternatives each, forward
        # only, an odd row count
        dict(name="linear_score_bf16", kind="linear", nodes=4099, rows=4099, width=1024, classes=50021, k=5, top=16,
             temperature=1.0, dtype="bf16", bias=True, grad=False, none=0.0),
        # one row of a vocabulary's logits
        dict(name="kept_one_f32", kind="kept", rows=1, classes=131072, k=1, top=8, temperature=0.7, dtype="f32",
             grad=False, none=0.0),
        # a mini-batch of the sampled configuration on kept logits
        dict(name="kept_batch_f32", kind="kept", rows=1024, classes=172, k=1, top=0, temperature=1.0, dtype="f32",
             grad=True, none=0.0),
        # a batch over a vocabulary, sixteen alternatives a row
        dict(name="kept_vocabulary_bf16", kind="kept", rows=8192, classes=50021, k=4, top=16, temperature=1.0,
             dtype="bf16", grad=False, none=0.0),
        # a training step on kept logits of a catalogue
        dict(name="kept_train_bf16", kind="kept", rows=4099, classes=100003, k=1, top=0, temperature=1.0,
             dtype="bf16", grad=True, none=0.1),
        # the parameters of a graph network of 608 features and hidden width 256
        dict(name="clip_graph_f32", kind="clip", tensors=8, most=608 * 256, dtype="f32", scaled=False),
        # those and a vocabulary's 16-bit classifier, under a loss scale
        dict(name="clip_vocabulary_bf16", kind="clip", tensors=9, most=131072 * 4096, dtype="bf16", scaled=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "kept", "kept", "clip"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "clip":
        return dict(kind=kind, tensors=_log(rng, 1, 400), most=_log(rng, 100, 50000000), dtype=dtype,
                    scaled=rng.random() < 0.5)
    classes = _log(rng, 47, 131072)
    grad = rng.random() < 0.6
    rows = _log(rng, 1, 30000)
    c = dict(kind=kind, classes=classes, k=rng.choice([1, 1, min(classes, _log(rng, 1, 64))]),
             temperature=rng.choice([0.7, 1.0, 1.0, 1.5]), dtype=dtype, grad=grad,
             top=0 if grad or rng.random() < 0.4 else min(classes, _log(rng, 1, 64)))
    if kind == "kept":
        c["rows"] = max(1, min(rows, 400000000 // classes))
    else:
        width = rng.choice([_log(rng, 16, 4096), 8 * _log(rng, 8, 512), 64 * _log(rng, 1, 64)])
        # at most a twentieth of the largest listed case's products in 16 bits
        c["rows"] = max(1, min(rows, (200000000000 if dtype != "f32" else 40000000000) // (width * classes),
                               400000000 // classes))
        c["nodes"] = c["rows"] if rng.random() < 0.5 else c["rows"] + rng.randint(0, c["rows"])
        c.update(width=width, bias=rng.random() < 0.5)
    c["none"] = rng.choice([0.0, 0.1, 0.5]) if c["rows"] > 64 else 0.0
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def _sizes(case):
    """Elements of the tensors: the largest first, the others anything below
    (weights and biases)."""
    rng = random.Random(case["tensors"])
    return [case["most"]] + [_log(rng, 1, case["most"] / 4) for _ in range(case["tensors"] - 1)]


def _on_grid(x, step):
    """x in whole steps of at most 127: what an 8-bit quantised operand holds."""
    return (x / step).round_().clamp_(-127, 127).mul_(step)


def prepare(case, seed):
    gen = _generator(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["kind"] == "clip":
        # tensors of one model have gradients of different sizes; together
        # their norm is 8 to 16 times what it may be
        sizes = _sizes(case)
        level = torch.exp(torch.randn(len(sizes), generator=gen, device=DEV))
        total = torch.sqrt(sum(n * l * l for n, l in zip(sizes, level)))
        up = 4096.0 if case["scaled"] else 1.0
        aim = 8.0 + 8.0 * torch.rand((), generator=gen, device=DEV)
        s["grads"] = [(torch.randn(n, generator=gen, device=DEV) * (l * aim * up / total)).to(dt)
                      for n, l in zip(sizes, level)]
        s["scale"] = torch.tensor(1.0 / up, device=DEV) if case["scaled"] else None
        s["out"] = [torch.empty(n, device=DEV) for n in sizes]
        return s
    n, classes, k = case["rows"], case["classes"], case["k"]
    lab = torch.randint(0, classes, (n,), generator=gen, device=DEV)
    if case["kind"] == "kept":
        # a model's logits: a bulk, and a few classes that stand out
        z = torch.randn(n, classes, generator=gen, device=DEV) * 2.0
        best = torch.randint(0, classes, (n, 4), generator=gen, device=DEV)
        best[:, 0] = lab
        z.scatter_add_(1, best, torch.full((n, 4), 6.0, device=DEV))
        s["logits"] = z.to(dt).requires_grad_(case["grad"])
    else:
        # rows of unit length: a hidden row is noise plus a multiple of its
        # class's row, so that its logit stands clear of the others (four rows
        # in five, as a trained model has it) or well below them
        nodes, width = case["nodes"], case["width"]
        w = torch.randn(classes, width, generator=gen, device=DEV) / math.sqrt(width)
        h = torch.randn(nodes, width, generator=gen, device=DEV)
        rows = None
        if nodes != n:
            rows = torch.sort(torch.randperm(nodes, generator=gen, device=DEV)[:n]).values
        high = math.sqrt(2.0 * math.log(classes))
        pull = torch.where(torch.rand(n, generator=gen, device=DEV) < 0.8, high + 6.0, high - 5.0)
        at = rows if rows is not None else torch.arange(n, device=DEV)
        h[at] += pull[:, None] * w[lab]
        b = 0.1 * torch.randn(classes, generator=gen, device=DEV) if case["bias"] else None
        if case["top"]:
            # Alternatives are told by their order, so the operands of these
            # cases are those of a classifier quantised to 8 bits: products
            # are whole multiples of a power of two and their sums below 2^24
            # of it, so a logit is one number in whatever order it is summed,
            # and equal ones go to the lowest class.
            w = _on_grid(w, 2.0 ** (math.ceil(math.log2(4.0 / math.sqrt(width))) - 7))
            h = _on_grid(h, 2.0 ** -4)
            b = _on_grid(b, 2.0 ** -6) if b is not None else None
        s["rows"] = rows
        s["hidden"] = h.to(dt).requires_grad_(case["grad"])
        s["weight"] = w.to(dt).requires_grad_(case["grad"])
        s["bias"] = b.to(dt).requires_grad_(case["grad"]) if b is not None else None
    # the given classes: the sampled answer, mostly the best one, and other
    # candidates; some places have none
    j = torch.arange(k, device=DEV)
    step = torch.randint(1, max(2, classes // k + 1), (n, 1), generator=gen, device=DEV)
    index = (lab[:, None] + j * step) % classes
    index[torch.rand(n, k, generator=gen, device=DEV) < case["none"]] = -1
    s["index"] = index[:, 0] if k == 1 else index
    if case["grad"]:
        # rewards over the rows' mean, and a small bonus for entropy; f16
        # gradients are taken of a scaled loss, as a GradScaler does
        up = 4096.0 if case["dtype"] == "f16" else 1.0
        s["dlogp"] = torch.randn(s["index"].shape, generator=gen, device=DEV) * (-up / n)
        s["dentropy"] = torch.full((n,), -0.01 * up / n, device=DEV)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return _own(s) if own else _plain(s)


def _params(s):
    if s["case"]["kind"] == "kept":
        return [s["logits"]]
    return [s["hidden"], s["weight"]] + ([s["bias"]] if s["bias"] is not None else [])


def _own(s):
    from graph_rws_amd.core import clip_grads
    from graph_rws_amd.layers import linear_log_probs, log_probs

    case = s["case"]
    if case["kind"] == "clip":
        return [clip_grads(s["grads"], 1.0, out=s["out"], scale=s["scale"])] + s["out"]
    if case["kind"] == "kept":
        got = log_probs(s["logits"], s["index"], temperature=case["temperature"], top=case["top"])
    else:
        got = linear_log_probs(s["hidden"], s["weight"], s["index"], bias=s["bias"], rows=s["rows"],
                               temperature=case["temperature"], top=case["top"])
    out = [got.logp.detach(), got.entropy.detach()]
    if case["top"]:
        out += [got.top_logp, got.top_index]
    if case["grad"]:
        out += list(torch.autograd.grad([got.logp, got.entropy], _params(s), [s["dlogp"], s["dentropy"]]))
    return out


def _plain(s):
    case = s["case"]
    if case["kind"] == "clip":
        scale = 1.0 if s["scale"] is None else s["scale"]
        squares = [(g.double() * scale).square().sum() for g in s["grads"]]
        norm = torch.stack(squares).sum().sqrt()
        keep = torch.clamp(1.0 / (norm + 1e-6), max=1.0) * scale
        return [norm.float()] + [o.copy_(g.float() * keep) for o, g in zip(s["out"], s["grads"])]
    dt, t = DTYPES[case["dtype"]], case["temperature"]
    if case["kind"] == "kept":
        z = s["logits"].detach().float()
    else:
        h = s["hidden"].detach()
        h = (h if s["rows"] is None else h[s["rows"]]).float()
        w = s["weight"].detach().float()
        z = h @ w.t()
        if s["bias"] is not None:
            z += s["bias"].detach().float()
    if case["top"]:
        best, top_index = torch.sort(z, dim=1, descending=True, stable=True)
        best, top_index = best[:, :case["top"]] / t, top_index[:, :case["top"]].int()
    z = z / t
    z -= z.max(1, keepdim=True).values if not case["top"] else best[:, :1]
    p = torch.exp(z)
    total = p.sum(1, keepdim=True)
    z -= torch.log(total)
    p /= total
    entropy = -(p * z).sum(1)
    index = s["index"] if s["index"].dim() == 2 else s["index"][:, None]
    given = index >= 0
    at = index.clamp(min=0)
    logp = torch.where(given, z.gather(1, at), 0.0)
    out = [logp.view(s["index"].shape), entropy]
    if case["top"]:
        out += [best - best[:, :1] - torch.log(total), top_index]
    if not case["grad"]:
        return out
    a = torch.where(given, s["dlogp"].view(index.shape), 0.0)
    z += entropy[:, None]
    z *= s["dentropy"][:, None]
    z += a.sum(1, keepdim=True)
    g = p.mul_(z).neg_()
    del z
    g.scatter_add_(1, at, a)
    g /= t
    if case["kind"] == "kept":
        return out + [g.to(dt)]
    dh = g @ w
    if s["rows"] is not None:
        dh = torch.zeros(s["hidden"].shape, device=DEV).index_copy(0, s["rows"], dh)
    out += [dh.to(dt), (g.t() @ h).to(dt)]
    if s["bias"] is not None:
        out.append(g.sum(0).to(dt))
    return out


# ---------------------------------------------------------------------------
# the least work, and results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "clip":
        n = sum(_sizes(case))
        return {"bytes": n * (e + 4), "flops": 3 * n}
    n, classes, k = case["rows"], case["classes"], case["k"]
    least = 8 * n * k + 4 * n * (k + 1) + 8 * n * case["top"]
    if case["grad"]:
        least += 4 * n * (k + 1)
    if case["kind"] == "kept":
        return {"bytes": least + n * classes * e * (2 if case["grad"] else 1), "flops": 4 * n * classes}
    width = case["width"]
    params = (classes * width + (classes if case["bias"] else 0)) * e
    least += n * width * e + params
    if case["grad"]:
        least += case["nodes"] * width * e + params
    return {"bytes": least, "flops": (3 if case["grad"] else 1) * 2 * n * width * classes}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "clip":
        grads = [g.double() for g in s["grads"]]
        if s["scale"] is not None:
            grads = [g / 4096.0 for g in grads]
        norm = math.sqrt(sum(float(torch.dot(g, g)) for g in grads))
        return [torch.tensor(norm, dtype=torch.float64, device=DEV)] + [g * min(1.0, 1.0 / (norm + 1e-6))
                                                                        for g in grads]
    if case["kind"] == "kept":
        x = None
        z = s["logits"].detach().double()
    else:
        w = s["weight"].detach().double()
        x = s["hidden"].detach().double()
        x = x if s["rows"] is None else x.index_select(0, s["rows"])
        z = torch.mm(x, w.t())
        if s["bias"] is not None:
            z.add_(s["bias"].detach().double())
    order = torch.argsort(-z, dim=1, stable=True)[:, :case["top"]] if case["top"] else None
    z.div_(case["temperature"])
    logq = torch.log_softmax(z, 1)
    del z
    q = torch.exp(logq)
    entropy = torch.special.entr(q).sum(1)
    index = s["index"].view(case["rows"], case["k"])
    logp = logq.gather(1, index.clamp(min=0)).masked_fill(index < 0, 0.0)
    out = [logp.view(s["index"].shape), entropy]
    if order is not None:
        out += [logq.gather(1, order), order.int()]
    if not case["grad"]:
        return out
    a = s["dlogp"].double().view(index.shape).masked_fill(index < 0, 0.0)
    # d entropy / d z = -q (log q + entropy); d logp_j / d z = [j] - q
    d = logq.add_(entropy[:, None]).mul_(s["dentropy"].double()[:, None])
    d.add_(a.sum(1)[:, None]).mul_(q).neg_()
    del q
    d.scatter_add_(1, index.clamp(min=0), a)
    d.div_(case["temperature"])
    if x is None:
        return out + [d]
    dh = torch.mm(d, w)
    if s["rows"] is not None:
        full = torch.zeros(s["hidden"].shape, dtype=torch.float64, device=DEV)
        full[s["rows"]] = dh
        dh = full
    out += [dh, torch.mm(d.t(), x)]
    if s["bias"] is not None:
        out.append(d.sum(0))
    return out
