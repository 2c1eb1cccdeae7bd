"""What a model of tokens trains with around its attention, as measurable cases: the
embedding lookup with its gradient, layer norm with its gradients, the loss of
token labels with its gradient, and the global norm of many gradients with their
clipping. Tensors are matrices of one row per token.

With `own` false, run() computes plain torch forms in float32; with `own` true
it makes the calls of ferrograd_amd (Tensor.embedding, Tensor.layer_norm,
Tensor.token_cross_entropy, clip_norm and Tensor.gradient). prepare() draws the
same inputs either way, on the GPU and from the seed alone; with `own` true it
uploads them as the framework's tensors, which is how a program of the framework
holds its data."""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5

# The parameters of a small token model: an embedding, two layers (of keys and values with a weight and a bias, queries,
# the projection back, two norms and an MLP of an odd width), and a last norm's weight and bias.
LAYER = "512x2048,512,2048x2048,2048x2048,2048,2048,8191x2048,8191,2048x8191"
MODEL = ",".join(["32000x2048", LAYER, LAYER, "2048", "2048"])


def listed():
    return [
        # The tokens of one step of eight sequences: launches and host latency.
        {"name": "embed_step_8x1024", "kind": "embedding", "tokens": 8, "vocab": 32000, "dim": 1024, "ids": "uniform",
         "grad": False},
        # A train batch of ragged sizes, tokens as frequent as words are, and the weight's gradient.
        {"name": "embed_grad_5001x777", "kind": "embedding", "tokens": 5001, "vocab": 20011, "dim": 777, "ids": "words",
         "grad": True},
        # A long train batch, a third of it one padding token, and the weight's gradient.
        {"name": "embed_grad_65536x2048", "kind": "embedding", "tokens": 65536, "vocab": 50001, "dim": 2048,
         "ids": "padded", "grad": True},
        # The hidden states of one step of eight sequences.
        {"name": "layer_norm_step_8x1024", "kind": "layer_norm", "rows": 8, "dim": 1024, "bias": True, "grad": False},
        # A train batch with an odd width: forward and the gradients of input, weight and bias.
        {"name": "layer_norm_grad_5001x777", "kind": "layer_norm", "rows": 5001, "dim": 777, "bias": True, "grad": True},
        # A long train batch of wide hidden states: forward and gradients.
        {"name": "layer_norm_grad_16384x4096", "kind": "layer_norm", "rows": 16384, "dim": 4096, "bias": True,
         "grad": True},
        # The loss of the 784-128-10 classifier at batch 256, by class labels, and the logits' gradient.
        {"name": "loss_grad_256x10", "kind": "loss", "rows": 256, "classes": 10, "banned": 0, "ignored": 0.0,
         "grad": True},
        # Scoring a few tokens under a large vocabulary: few long rows.
        {"name": "loss_8x128000", "kind": "loss", "rows": 8, "classes": 128000, "banned": 0, "ignored": 0.0,
         "grad": False},
        # A train batch whose vocabulary is padded with columns of -inf, some labels ignored.
        {"name": "loss_grad_2047x50001", "kind": "loss", "rows": 2047, "classes": 50001, "banned": 47, "ignored": 0.2,
         "grad": True},
        # A long train batch under an ordinary vocabulary.
        {"name": "loss_grad_8192x32000", "kind": "loss", "rows": 8192, "classes": 32000, "banned": 0, "ignored": 0.1,
         "grad": True},
        # The gradients of the 784-128-10 classifier.
        {"name": "clip_classifier", "kind": "clip", "shapes": "128x784,128,10x128,10", "size": 0.01, "max_norm": 1.0},
        # The gradients of a small token model, large and tiny tensors among them.
        {"name": "clip_model", "kind": "clip", "shapes": MODEL, "size": 0.001, "max_norm": 1.0},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embedding", "layer_norm", "loss", "clip"])
    case = {"kind": kind}
    if kind == "embedding":
        case["dim"] = _log_int(rng, 1, 4096)
        case["tokens"] = min(_log_int(rng, 1, 1 << 17), (1 << 26) // case["dim"])
        case["vocab"] = min(_log_int(rng, 2, 200000), (1 << 26) // case["dim"])
        case["ids"] = rng.choice(["uniform", "words", "words", "padded", "outside", "one"])
    elif kind == "layer_norm":
        # From 4 columns on: the gradient of two is what float32 leaves of a difference.
        case["dim"] = _log_int(rng, 4, 20000)
        case["rows"] = min(_log_int(rng, 1, 1 << 17), (1 << 25) // case["dim"])
        case["bias"] = rng.random() < 0.7
    elif kind == "loss":
        case["classes"] = _log_int(rng, 2, 130000)
        case["rows"] = min(_log_int(rng, 1, 1 << 17), (1 << 27) // case["classes"])
        case["banned"] = rng.choice([0, 0, case["classes"] // 3])
        case["ignored"] = rng.choice([0.0, 0.0, 0.1, 0.5, 1.0])
    else:
        count = _log_int(rng, 1, 60)
        sizes = [_log_int(rng, 1, (1 << 27) // count) for _ in range(count)]
        case["shapes"] = ",".join(str(n) for n in sizes)
        # The norm is near size times the root of all elements: clipped or not, from tiny to large gradients.
        case["size"] = rng.choice([1e-4, 0.01, 1.0, 100.0])
        case["max_norm"] = round(case["size"] * math.sqrt(sum(sizes)) * rng.choice([0.01, 0.5, 3.0]), 6) or 1.0
    if kind != "clip":
        case["grad"] = rng.random() < 0.6
    return case


# ── inputs, from the seed alone ─────────────────────────────────────────────


def _shapes(case):
    return [[int(n) for n in s.split("x")] for s in case["shapes"].split(",")]


def _inputs(case, seed):
    """The case's tensors by name (clip's gradients as a list); whole numbers are int32."""
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(n):
        return torch.rand(n, generator=g, device="cuda", dtype=torch.float64)

    if case["kind"] == "embedding":
        t, v = case["tokens"], case["vocab"]
        u, share = uniform(t), uniform(t)
        even = (u * v).long().clamp(max=v - 1)
        # Words: the k-th most frequent of them is 1/k as frequent as the first, under ids in any order.
        ranked = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp(0, v - 1)
        ids = torch.randperm(v, generator=g, device="cuda")[ranked] if case["ids"] in ("words", "padded") else even
        if case["ids"] == "padded":
            ids = torch.where(share < 1 / 3, 0, ids)
        elif case["ids"] == "outside":  # padding that is no token
            ids = torch.where(share < 1 / 3, torch.where(share < 1 / 4, -1, v), ids)
        elif case["ids"] == "one":
            ids = ids[:1].expand(t)
        got = {"weight": 0.05 * normal(v, case["dim"]), "ids": ids.to(torch.int32).contiguous()}
        if case["grad"]:
            got["g"] = normal(t, case["dim"])
        return got
    if case["kind"] == "layer_norm":
        n, d = case["rows"], case["dim"]
        got = {"x": 2.0 + 3.0 * normal(n, d), "weight": 1.0 + 0.1 * normal(d)}
        if case["bias"]:
            got["bias"] = 0.1 * normal(d)
        if case["grad"]:
            got["g"] = normal(n, d)
        return got
    if case["kind"] == "loss":
        n, c, real = case["rows"], case["classes"], case["classes"] - case["banned"]
        # Logits of a few units, and the label's raised as by training.
        logits = 3.0 * normal(n, c)
        labels = (uniform(n) * real).long().clamp(max=real - 1)
        at = torch.arange(n, device="cuda")
        logits[at, labels] += 4.0
        logits[:, real:] = -math.inf
        labels = torch.where(uniform(n) < case["ignored"], -1, labels)
        return {"logits": logits, "labels": labels.to(torch.int32)}
    return {"grads": [case["size"] * normal(*s) for s in _shapes(case)]}


LEAVES = {"embedding": ["weight"], "layer_norm": ["x", "weight", "bias"], "loss": ["logits"]}


def _scale(case):
    """What an embedding's rows are scaled by: the root of their width."""
    return math.sqrt(case["dim"])


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        import ferrograd_amd as fg

        def upload(x):
            return fg.Tensor.new(x.cpu().numpy(), list(x.shape), "hip")

        for name, x in list(state.items()):
            if name == "grads":
                state[name] = [upload(t) for t in x]
            elif torch.is_tensor(x):
                state[name] = upload(x)
                if case["grad"] and name in LEAVES[case["kind"]]:
                    state[name].with_requires_grad(True)
        fg.synchronize("hip")
    return state


# ── the framework's calls ───────────────────────────────────────────────────


class _Buffer:
    """A realised tensor's device buffer, for torch to view; keeps the tensor."""

    def __init__(self, t):
        self.t = t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": "<f4", "data": (t.data_ptr()[0], False),
                                         "version": 2}


def _view(t):
    return torch.as_tensor(_Buffer(t), device="cuda")


def _own_run(s):
    import ferrograd_amd as fg

    case = s["case"]
    if case["kind"] == "clip":
        norm, clipped = fg.clip_norm(s["grads"], case["max_norm"])
        fg.Tensor.realize_many([norm] + clipped)
        return {"norm": _view(norm), "clipped": [_view(t) for t in clipped]}
    if case["kind"] == "loss":
        outs = {"loss": s["logits"].token_cross_entropy(s["labels"])}
        if case["grad"]:
            outs["dlogits"] = outs["loss"].gradient([s["logits"]])[0]
    else:
        if case["kind"] == "embedding":
            y = s["weight"].embedding(s["ids"], scale=_scale(case))
        else:
            y = s["x"].layer_norm(s["weight"], s.get("bias"), eps=EPS)
        outs = {"y": y}
        if case["grad"]:
            wrt = [name for name in LEAVES[case["kind"]] if name in s]
            grads = y.mul(s["g"]).sum([0, 1]).gradient([s[name] for name in wrt])
            outs.update({"d" + name: g for name, g in zip(wrt, grads)})
    fg.Tensor.realize_many(list(outs.values()))
    return {name: _view(t) for name, t in outs.items()}


# ── the plain forms ─────────────────────────────────────────────────────────


def _plain_embedding(case, s):
    """Rows of the weight by id, scaled; ids outside of the weight are rows of zeros and have no gradient."""
    inside = ((s["ids"] >= 0) & (s["ids"] < case["vocab"]))[:, None]
    at = s["ids"].clamp(0, case["vocab"] - 1).long()
    outs = {"y": torch.where(inside, s["weight"][at] * _scale(case), 0.0)}
    if case["grad"]:
        outs["dweight"] = torch.zeros_like(s["weight"]).index_add_(0, at, torch.where(inside, s["g"], 0.0)) * _scale(case)
    return outs


def _plain_layer_norm(case, s):
    x, w = s["x"], s["weight"]
    centred = x - x.mean(1, keepdim=True)
    inv = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
    normed = centred * inv
    y = normed * w
    outs = {"y": y + s["bias"] if case["bias"] else y}
    if case["grad"]:
        gw = s["g"] * w
        outs["dx"] = inv * (gw - gw.mean(1, keepdim=True) - normed * (gw * normed).mean(1, keepdim=True))
        outs["dweight"] = (s["g"] * normed).sum(0)
        if case["bias"]:
            outs["dbias"] = s["g"].sum(0)
    return outs


def _plain_loss(case, s):
    """The mean of logsumexp(row) - row[label] over the rows whose label is a class."""
    x, labels = s["logits"], s["labels"].long()
    valid = (labels >= 0) & (labels < case["classes"])
    count = valid.sum().clamp(min=1)
    at = torch.where(valid, labels, 0)[:, None]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    each = torch.where(valid, (top + torch.log(total) - x.gather(1, at))[:, 0], 0.0)
    outs = {"loss": (each.double().sum() / count).float().reshape(1)}
    if case["grad"]:
        p = e / total
        p.scatter_add_(1, at, torch.full_like(top, -1.0))
        outs["dlogits"] = torch.where(valid[:, None], p / count, 0.0)
    return outs


def _plain_clip(case, s):
    """x max_norm / max(norm, max_norm) of every tensor, norm the root of the sum of all squares."""
    norm = torch.stack([(t * t).sum() for t in s["grads"]]).double().sum().sqrt()
    scale = (case["max_norm"] / norm.clamp(min=case["max_norm"])).float()
    return {"norm": norm.float().reshape(1), "clipped": [t * scale for t in s["grads"]]}


PLAIN = {"embedding": _plain_embedding, "layer_norm": _plain_layer_norm, "loss": _plain_loss, "clip": _plain_clip}


def run(s):
    if own:
        return _own_run(s)
    return PLAIN[s["case"]["kind"]](s["case"], s)


# ── what a pass cannot do without ───────────────────────────────────────────


def work(case):
    """Each input read once (of an embedding's weight the rows that differ, at most one a token), each output written
    once."""
    grad = case.get("grad", False)
    if case["kind"] == "embedding":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        floats = (min(n, v) + n + n / d + (n + n / d + v if grad else 0)) * d
        return {"bytes": int(4 * floats), "flops": (2 if grad else 1) * n * d}
    if case["kind"] == "layer_norm":
        n, d = case["rows"] * case["dim"], case["dim"]
        vectors = 1 + case["bias"]
        return {"bytes": int(4 * ((4 if grad else 2) * n + vectors * (2 if grad else 1) * d)), "flops": (20 if grad else 8) * n}
    if case["kind"] == "loss":
        n = case["rows"] * case["classes"]
        return {"bytes": 4 * ((2 if grad else 1) * n + case["rows"] + 1), "flops": (6 if grad else 4) * n}
    n = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": 8 * n + 4, "flops": 3 * n}


# ── the same in 64 bits ─────────────────────────────────────────────────────


def _exact_embedding(case, d):
    ids, table = d["ids"].long(), torch.zeros(case["vocab"] + 1, case["dim"], dtype=torch.float64, device="cuda")
    table[:-1] = d["weight"].double() * case["dim"] ** 0.5
    ids = torch.where((ids < 0) | (ids >= case["vocab"]), case["vocab"], ids)  # the last row is of zeros
    outs = {"y": table[ids]}
    if case["grad"]:
        # Tokens sorted by id: the difference of the running sums at an id's ends.
        order = torch.argsort(ids, stable=True)
        ends = torch.bincount(ids, minlength=case["vocab"] + 1).cumsum(0)
        outs["dweight"] = torch.empty(case["vocab"], case["dim"], dtype=torch.float64, device="cuda")
        for c in range(0, case["dim"], 256):
            sums = torch.zeros(case["tokens"] + 1, min(256, case["dim"] - c), dtype=torch.float64, device="cuda")
            sums[1:] = d["g"][:, c:c + 256].double()[order].cumsum(0)
            upto = sums[ends]
            part = upto[:-1].clone()
            part[1:] -= upto[:-2]
            outs["dweight"][:, c:c + 256] = part * case["dim"] ** 0.5
    return outs


def _exact_layer_norm(case, d):
    leaves = {n: d[n].double().requires_grad_(case["grad"]) for n in ("x", "weight", "bias") if n in d}
    var, mean = torch.var_mean(leaves["x"], 1, correction=0, keepdim=True)
    y = (leaves["x"] - mean) / (var + EPS).sqrt() * leaves["weight"] + leaves.get("bias", 0.0)
    if not case["grad"]:
        return {"y": y}
    grads = torch.autograd.grad(y, list(leaves.values()), d["g"].double())
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}


def _exact_loss(case, d):
    labels = d["labels"].long()
    kept = ((labels >= 0) & (labels < case["classes"])).nonzero()[:, 0]
    total = torch.zeros(1, dtype=torch.float64, device="cuda")
    grads = torch.zeros(case["rows"], case["classes"], dtype=torch.float64, device="cuda") if case["grad"] else None
    for rows in kept.split(1024):
        logp = torch.log_softmax(d["logits"][rows].double(), 1)
        picked = torch.arange(len(rows), device="cuda"), labels[rows]
        total -= logp[picked].sum()
        if case["grad"]:
            p = logp.exp()
            p[picked] = torch.expm1(logp[picked])
            grads[rows] = p / len(kept)
    outs = {"loss": total / max(1, len(kept))}
    return {**outs, "dlogits": grads} if case["grad"] else outs


def _exact_clip(case, d):
    norm = math.sqrt(sum(float(torch.dot(t.reshape(-1).double(), t.reshape(-1).double())) for t in d["grads"]))
    scale = min(1.0, case["max_norm"] / norm) if norm > 0 else 1.0
    return {"norm": torch.tensor([norm], dtype=torch.float64, device="cuda"), "clipped": [t.double() * scale for t in d["grads"]]}


def exact(case, seed):
    d = _inputs(case, seed)
    return {"embedding": _exact_embedding, "layer_norm": _exact_layer_norm, "loss": _exact_loss, "clip": _exact_clip}[
        case["kind"]](case, d)
