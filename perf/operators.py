"""Attention with its gradients, per-head norms with the position rotation, and
dropout, as measurable cases. Tensors are matrices of one row per token, as
Linear takes and gives them: queries [batch * length, heads * head_dim].

With `own` false, run() computes plain torch forms in float32; with `own` true
it makes the calls of ferrograd_amd (Tensor.attention, Tensor.norm_rotate,
Tensor.dropout and Tensor.gradient). prepare() draws the same inputs either
way, on the GPU and from the seed alone; with `own` true it uploads them as the
framework's tensors, which is how a program of the framework holds its data."""
from __future__ import annotations

import math

import torch

own = False

LARGEST_PAIRS = 8192 * 8192 * 16 * 128  # query-key pairs times head_dim of the largest attention case


def listed():
    return [
        # Attention of a few short sequences: the smallest calls, launches and host latency.
        {"name": "attend_tiny", "kind": "attention", "batch": 2, "sq": 33, "sk": 33, "heads": 4, "kv_heads": 4,
         "dim": 32, "causal": True, "lengths": False, "grad": False},
        # A prompt through grouped heads, as a model that answers reads it.
        {"name": "attend_prompt_4096", "kind": "attention", "batch": 1, "sq": 4096, "sk": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "causal": True, "lengths": False, "grad": False},
        # One new token for each of eight sequences over long contexts of their own lengths.
        {"name": "attend_token_8192", "kind": "attention", "batch": 8, "sq": 1, "sk": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "causal": False, "lengths": True, "grad": False},
        # A train step's attention over short sequences: forward and the gradients of q, k and v.
        {"name": "attend_grad_256", "kind": "attention", "batch": 8, "sq": 256, "sk": 256, "heads": 8, "kv_heads": 8,
         "dim": 64, "causal": True, "lengths": False, "grad": True},
        # A padded batch with ragged sides, both directions visible (an encoder), and its gradients.
        {"name": "attend_grad_ragged", "kind": "attention", "batch": 5, "sq": 777, "sk": 777, "heads": 12,
         "kv_heads": 12, "dim": 80, "causal": False, "lengths": True, "grad": True},
        # A train step over a long sequence: forward and gradients.
        {"name": "attend_grad_8192", "kind": "attention", "batch": 1, "sq": 8192, "sk": 8192, "heads": 16,
         "kv_heads": 4, "dim": 128, "causal": True, "lengths": False, "grad": True},
        # The queries of one token per sequence, far into their contexts.
        {"name": "norm_rotate_8x32x128", "kind": "norm_rotate", "tokens": 8, "heads": 32, "dim": 128,
         "base": 500000.0, "far": 1 << 20, "grad": False},
        # The keys of a batch with an odd head size: forward and gradients.
        {"name": "norm_rotate_grad_5001x7x74", "kind": "norm_rotate", "tokens": 5001, "heads": 7, "dim": 74,
         "base": 10000.0, "far": 5001, "grad": True},
        # The queries of a long train batch: forward and gradients.
        {"name": "norm_rotate_grad_16384x32x128", "kind": "norm_rotate", "tokens": 16384, "heads": 32, "dim": 128,
         "base": 500000.0, "far": 16384, "grad": True},
        # The hidden layer of the 784-128-10 classifier at batch 256.
        {"name": "dropout_256x128", "kind": "dropout", "rows": 256, "cols": 128, "p": 0.5, "grad": False},
        # The hidden layer of a wide MLP with an odd width: forward and gradient.
        {"name": "dropout_grad_8192x4001", "kind": "dropout", "rows": 8192, "cols": 4001, "p": 0.1, "grad": True},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "norm_rotate", "dropout"])
    case = {"kind": kind, "grad": rng.random() < 0.6}
    if kind == "attention":
        kv_heads = _log_int(rng, 1, 16)
        case["heads"], case["kv_heads"] = kv_heads * rng.choice([1, 1, 2, 4, 5]), kv_heads
        case["dim"] = rng.choice([16, 32, 40, 64, 64, 72, 80, 96, 100, 128, 128, rng.randint(8, 128)])
        case["batch"] = _log_int(rng, 1, 8)
        how = rng.choice(["self", "self", "self", "token", "cross"])
        case["sk"] = _log_int(rng, 1, 16384 if how == "token" else 6000)
        case["sq"] = {"self": case["sk"], "token": 1, "cross": _log_int(rng, 1, 3000)}[how]
        case["causal"] = how == "self" and rng.random() < 0.7 or how == "cross" and rng.random() < 0.3
        case["lengths"] = rng.random() < 0.5
        case["grad"] = case["grad"] and how != "token"
        while (case["batch"] * case["sq"] * case["sk"] * case["heads"] * case["dim"] > LARGEST_PAIRS // 2
               or case["batch"] * case["sk"] * case["kv_heads"] * case["dim"] > 8 * 8192 * 8 * 128):
            side = "batch" if case["batch"] > 1 else "sk"
            case[side] = max(1, case[side] // 2)
            case["sq"] = case["sk"] if how == "self" else case["sq"]
    elif kind == "norm_rotate":
        case["heads"], case["dim"] = _log_int(rng, 1, 40), 2 * _log_int(rng, 4, 128)
        case["tokens"] = min(_log_int(rng, 1, 32768), (1 << 26) // (case["heads"] * case["dim"]))
        case["base"] = rng.choice([10000.0, 500000.0, 1e6])
        case["far"] = max(case["tokens"], _log_int(rng, 16, 1 << 20))
    else:
        n = _log_int(rng, 1, 1 << 25)
        case["rows"] = _log_int(rng, 1, n)
        case["cols"], case["p"] = max(1, n // case["rows"]), rng.choice([0.0, 0.1, 0.2, 0.5, round(rng.random(), 3)])
    return case


# ── inputs, from the seed alone ─────────────────────────────────────────────


def _inputs(case, seed):
    """The case's tensors by name; whole-number inputs are int32."""
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def integers(lo, hi, n):
        return torch.randint(lo, hi, (n,), generator=g, device="cuda", dtype=torch.int32)

    if case["kind"] == "attention":
        b, d = case["batch"], case["dim"]
        rows_q, rows_k, hq, hk = b * case["sq"], b * case["sk"], case["heads"] * d, case["kv_heads"] * d
        # Queries of normed heads times a learned gain: scores of a few units, peaked softmax rows among flat ones.
        got = {"q": 2.0 * normal(rows_q, hq), "k": normal(rows_k, hk), "v": normal(rows_k, hk)}
        if case["grad"]:
            got["g"] = normal(rows_q, hq)
        if case["lengths"]:
            got["lengths"] = integers(1, case["sk"] + 1, b)
        return got
    if case["kind"] == "norm_rotate":
        t, w = case["tokens"], case["heads"] * case["dim"]
        got = {"x": 3.0 * normal(t, w), "weight": 1.0 + 0.1 * normal(case["dim"]),
               "positions": integers(0, case["far"], t)}
        if case["grad"]:
            got["g"] = normal(t, w)
        return got
    got = {"x": normal(case["rows"], case["cols"])}
    if case["grad"]:
        got["g"] = normal(case["rows"], case["cols"])
    return got


EPS = 1e-6


def _seed_of(seed):
    """Dropout's seed and offset: 64 bits of seed, a step count as offset."""
    return (int(seed) * 0x9E3779B97F4A7C15 + 0x632BE59BD9B4E019) % (1 << 63), int(seed) % 100000


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if case["kind"] == "dropout":
        state["seed"], state["offset"] = _seed_of(seed)
    if own:
        import ferrograd_amd as fg

        for name, x in list(state.items()):
            if torch.is_tensor(x):
                t = state[name] = fg.Tensor.new(x.cpu().numpy(), list(x.shape), "hip")
                if case["grad"] and name in ("q", "k", "v", "x", "weight"):
                    t.with_requires_grad(True)
        fg.synchronize("hip")
    return state


# ── the framework's calls ───────────────────────────────────────────────────


class _Buffer:
    """A realised tensor's device buffer, for torch to view; keeps the tensor."""

    def __init__(self, t):
        self.t = t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": "<f4", "data": (t.data_ptr()[0], False),
                                         "version": 2}


def _own_run(s):
    from ferrograd_amd import Tensor

    case = s["case"]
    if case["kind"] == "attention":
        wrt = ["q", "k", "v"]
        y = s["q"].attention(s["k"], s["v"], heads=case["heads"], kv_heads=case["kv_heads"], batch=case["batch"],
                             causal=case["causal"], lengths=s.get("lengths"))
    elif case["kind"] == "norm_rotate":
        wrt = ["x", "weight"]
        y = s["x"].norm_rotate(s["weight"], s["positions"], heads=case["heads"], eps=EPS, base=case["base"])
    else:
        wrt = ["x"]
        y = s["x"].dropout(case["p"], s["seed"], s["offset"])
    outs = {"y": y}
    if case["grad"]:
        grads = y.mul(s["g"]).sum([0, 1]).gradient([s[name] for name in wrt])
        outs.update({"d" + name: g for name, g in zip(wrt, grads)})
    Tensor.realize_many(list(outs.values()))
    return {name: torch.as_tensor(_Buffer(t), device="cuda") for name, t in outs.items()}


# ── the plain forms ─────────────────────────────────────────────────────────


def _heads(x, batch, heads):
    """[batch * length, heads * dim] as [batch, heads, length, dim]."""
    return x.reshape(batch, -1, heads, x.shape[1] // heads).permute(0, 2, 1, 3)


def _rows(x):
    """[batch, heads, length, dim] back as [batch * length, heads * dim]."""
    b, h, n, d = x.shape
    return x.permute(0, 2, 1, 3).reshape(b * n, h * d)


def _visible(case, lengths, device):
    """[batch, 1, sq, sk]: which keys each query sees."""
    i = torch.arange(case["sq"], device=device)[:, None]
    j = torch.arange(case["sk"], device=device)[None, :]
    seen = (j >= 0) if lengths is None else j < lengths[:, None, None, None]
    if case["causal"]:
        seen = seen & (j <= i + (case["sk"] - case["sq"]))
    return seen.expand(1 if lengths is None else len(lengths), 1, case["sq"], case["sk"])


def _plain_attention(case, s):
    group = case["heads"] // case["kv_heads"]
    scale = 1.0 / math.sqrt(case["dim"])
    q = _heads(s["q"], case["batch"], case["heads"])
    k, v = (_heads(s[n], case["batch"], case["kv_heads"]).repeat_interleave(group, 1) for n in "kv")
    seen = _visible(case, s.get("lengths"), q.device)
    scores = torch.where(seen, torch.matmul(q, k.transpose(2, 3)) * scale, -math.inf)
    top = scores.amax(3, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(3, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    y = torch.matmul(p, v)
    if not case["grad"]:
        return {"y": _rows(y)}
    g = _heads(s["g"], case["batch"], case["heads"])
    dv = torch.matmul(p.transpose(2, 3), g)
    ds = p * (torch.matmul(g, v.transpose(2, 3)) - (g * y).sum(3, keepdim=True)) * scale
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
    dk, dv = (x.reshape(case["batch"], case["kv_heads"], group, case["sk"], case["dim"]).sum(2) for x in (dk, dv))
    return {"y": _rows(y), "dq": _rows(dq), "dk": _rows(dk), "dv": _rows(dv)}


def _plain_norm_rotate(case, s):
    t, h, d = case["tokens"], case["heads"], case["dim"]
    # Far positions times a frequency: the angle needs 64 bits.
    freq = torch.exp(torch.arange(0, d, 2, device="cuda", dtype=torch.float64) * (-math.log(case["base"]) / d))
    angle = s["positions"].double()[:, None] * freq
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    x = s["x"].reshape(t, h, d)
    inv = torch.rsqrt((x * x).mean(2, keepdim=True) + EPS)
    normed = x * inv
    a, b = (normed * s["weight"]).chunk(2, 2)
    y = torch.cat([a * cos - b * sin, b * cos + a * sin], 2)
    if not case["grad"]:
        return {"y": y.reshape(t, h * d)}
    ga, gb = s["g"].reshape(t, h, d).chunk(2, 2)
    g = torch.cat([ga * cos + gb * sin, gb * cos - ga * sin], 2)
    gw = g * s["weight"]
    dx = inv * (gw - normed * (gw * normed).mean(2, keepdim=True))
    return {"y": y.reshape(t, h * d), "dx": dx.reshape(t, h * d), "dweight": (g * normed).sum((0, 1))}


# The constants of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011).
M0, M1, W0, W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
LOW = 0xFFFFFFFF


def _philox(n, seed, offset):
    """The first n random words (0 <= word < 2^32, as int64): word e is word e % 4 of the block with the counter
    (e // 4, offset) under the key `seed`, each 64 bits as (low, high) words."""
    block = torch.arange((n + 3) // 4, device="cuda")
    c0, c1 = block & LOW, block >> 32
    c2, c3 = torch.full_like(c0, offset & LOW), torch.full_like(c0, offset >> 32)
    k0, k1 = seed & LOW, seed >> 32
    for _ in range(10):
        x, y = c0 * M0, c2 * M1  # modulo 2^64; the shift's sign bits are masked away
        c0, c1, c2, c3 = ((y >> 32) & LOW) ^ c1 ^ k0, y & LOW, ((x >> 32) & LOW) ^ c3 ^ k1, x & LOW
        k0, k1 = (k0 + W0) & LOW, (k1 + W1) & LOW
    return torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:n]


def _plain_dropout(case, s):
    x, p = s["x"], case["p"]
    keep = (_philox(x.numel(), s["seed"], s["offset"]) >= int(p * 4294967296.0)).reshape(x.shape)
    scale = 1.0 / (1.0 - p)
    outs = {"y": torch.where(keep, x * scale, 0.0)}
    if case["grad"]:
        outs["dx"] = torch.where(keep, s["g"] * scale, 0.0)
    return outs


def run(s):
    if own:
        return _own_run(s)
    case = s["case"]
    plain = {"attention": _plain_attention, "norm_rotate": _plain_norm_rotate, "dropout": _plain_dropout}
    return plain[case["kind"]](case, s)


# ── what a pass cannot do without ───────────────────────────────────────────


def work(case):
    """Each input read once, each output written once; products over the visible pairs (of full lengths: half the
    longest on the average, where the sequences have lengths of their own)."""
    if case["kind"] == "attention":
        b, sq, sk, d = case["batch"], case["sq"], case["sk"], case["dim"]
        q, k = b * sq * case["heads"] * d, b * sk * case["kv_heads"] * d
        part = 0.5 if case["lengths"] else 1.0
        pairs = b * case["heads"] * part * sq * sk
        if case["causal"]:
            pairs = b * case["heads"] * sum(min(sk * part, max(0, i + 1 + sk - sq)) for i in range(sq))
        if not case["grad"]:
            return {"bytes": int(4 * (2 * q + 2 * part * k)), "flops": int(4 * pairs * d)}
        # Backward: the scores again, and the products for dv, dp, dq and dk.
        return {"bytes": int(4 * (4 * q + (2 + 2 * part) * k)), "flops": int(14 * pairs * d)}
    n = case["tokens"] * case["heads"] * case["dim"] if case["kind"] == "norm_rotate" else case["rows"] * case["cols"]
    streams = 4 if case["grad"] else 2
    if case["kind"] == "norm_rotate":
        return {"bytes": 4 * streams * n + 4 * case["tokens"] + 8 * case["dim"], "flops": (22 if case["grad"] else 8) * n}
    return {"bytes": 4 * streams * n, "flops": streams // 2 * n}


# ── the same in 64 bits ─────────────────────────────────────────────────────


def _exact_attention(case, d):
    b, hq, hk, dim = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    parts = {n: d[n].double().reshape(b, -1, hk if n in "kv" else hq, dim) for n in "qkvg" if n in d}
    outs = {"y": torch.zeros_like(parts["q"])}
    if case["grad"]:
        outs.update({"d" + n: torch.zeros_like(parts[n]) for n in "qkv"})
    for i in range(b):
        length = int(d["lengths"][i]) if "lengths" in d else case["sk"]
        hidden = None
        if case["causal"]:
            hidden = torch.ones(case["sq"], length, dtype=torch.bool, device="cuda").triu(1 + case["sk"] - case["sq"])
        for h in range(hq):
            at = h // (hq // hk)
            q = parts["q"][i, :, h].clone().requires_grad_(case["grad"])
            k, v = (parts[n][i, :length, at].clone().requires_grad_(case["grad"]) for n in "kv")
            scores = q @ k.T / math.sqrt(dim)
            if hidden is not None:
                scores = scores.masked_fill(hidden, -math.inf)
            probs = torch.softmax(scores, 1)
            if hidden is not None:
                probs = probs.masked_fill(hidden.all(1, keepdim=True), 0.0)
            y = probs @ v
            outs["y"][i, :, h] = y.detach()
            if case["grad"]:
                dq, dk, dv = torch.autograd.grad(y, [q, k, v], parts["g"][i, :, h])
                outs["dq"][i, :, h] = dq
                outs["dk"][i, :length, at] += dk
                outs["dv"][i, :length, at] += dv
    return {n: x.reshape(x.shape[0] * x.shape[1], -1) for n, x in outs.items()}


def _exact_norm_rotate(case, d):
    t, h, dim = case["tokens"], case["heads"], case["dim"]
    x, w = d["x"].double().requires_grad_(case["grad"]), d["weight"].double().requires_grad_(case["grad"])
    z = x.reshape(t, h, dim)
    z = z / ((z.square().sum(2, keepdim=True) / dim + EPS).sqrt()) * w
    # The pair (i, i + dim/2) as a complex number, turned by its angle.
    turn = d["positions"].double()[:, None] / case["base"] ** (torch.arange(dim // 2, device="cuda").double() * 2 / dim)
    turned = torch.complex(z[..., :dim // 2], z[..., dim // 2:]) * torch.polar(torch.ones_like(turn), turn)[:, None]
    y = torch.cat([turned.real, turned.imag], 2).reshape(t, h * dim)
    if not case["grad"]:
        return {"y": y}
    dx, dw = torch.autograd.grad(y, [x, w], d["g"].double())
    return {"y": y.detach(), "dx": dx, "dweight": dw}


def _exact_dropout(case, d, seed):
    key, offset = _seed_of(seed)
    n = case["rows"] * case["cols"]

    def times(a, m):  # (high, low) words of a 32 by 32 bit product, through 16-bit halves
        low, high = a * (m & 0xFFFF), a * (m >> 16)
        high = high + (low >> 16)
        return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)

    at = torch.arange(-(-n // 4), device="cuda")
    c = [at % (1 << 32), at // (1 << 32), torch.zeros_like(at) + offset % (1 << 32), torch.zeros_like(at) + (offset >> 32)]
    for r in range(10):
        ka, kb = (key % (1 << 32) + r * W0) % (1 << 32), ((key >> 32) + r * W1) % (1 << 32)
        h0, l0 = times(c[0], M0)
        h1, l1 = times(c[2], M1)
        c = [h1 ^ c[1] ^ ka, l1, h0 ^ c[3] ^ kb, l0]
    words = torch.stack(c, 1).reshape(-1)[:n].reshape(case["rows"], case["cols"])
    kept = (words >= int(case["p"] * 4294967296.0)).double() / (1.0 - case["p"])
    return {out: d[name].double() * kept for out, name in (("y", "x"), ("dx", "g")) if name in d}


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, d)
    if case["kind"] == "norm_rotate":
        return _exact_norm_rotate(case, d)
    return _exact_dropout(case, d, seed)
