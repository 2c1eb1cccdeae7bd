"""Attention, per-head norms with the position rotation, and dropout: refusals,
plans, values against float64, gradients against their formulas and against
differences, and runs of them together."""
import numpy as np
import pytest

import attention_ref
from attention_ref import U
from conftest import graphs_on, seeded


# ── refusals and plans (no GPU) ─────────────────────────────────────────────


def cpu_tensor(fg, shape, dtype=np.float32):
    return fg.Tensor.new(np.zeros(shape, dtype), list(shape), "cpu")


def test_attention_refusals(fg, cpu):
    t = lambda *s: cpu_tensor(fg, s)  # noqa: E731
    q, k = t(6, 16), t(10, 8)
    with pytest.raises(fg.FerrogradError, match="the cpu device has no kernel"):
        q.attention(k, k, heads=4, kv_heads=2, batch=2)
    for bad, kw, match in [
        ((k, k), dict(heads=4, kv_heads=2, batch=4), "do not split into a batch"),
        ((k, k), dict(heads=4, kv_heads=3, batch=2), "do not share 3 key heads evenly"),
        ((k, k), dict(heads=5, kv_heads=5, batch=2), "do not split into 5 heads"),
        ((k, k), dict(heads=4, kv_heads=4, batch=2), "k must have 4 heads of 4"),
        ((k, t(10, 4)), dict(heads=4, kv_heads=2, batch=2), "v must have k's shape"),
        ((t(10, 2, 4), k), dict(heads=4, kv_heads=2, batch=2), "k must be 2D"),
        ((cpu_tensor(fg, (10, 8), np.int32), k), dict(heads=4, kv_heads=2, batch=2), "k must be f32"),
        ((k, k), dict(heads=4, kv_heads=2, batch=2, lengths=t(2)), "lengths must be i32"),
        ((k, k), dict(heads=4, kv_heads=2, batch=2, lengths=cpu_tensor(fg, (3,), np.int32)), "lengths must be i32 of shape"),
        ((k, k), dict(heads=4, kv_heads=2, batch=2, scale=float("nan")), "scale must be finite"),
        ((k, k), dict(heads=0, kv_heads=2, batch=2), "at least 1"),
        ((k, k), dict(heads=4, kv_heads=2, batch=0), "at least 1"),
    ]:
        with pytest.raises(fg.FerrogradError, match=match):
            q.attention(*bad, **kw)
    with pytest.raises(fg.FerrogradError, match="at most 128, got 129"):
        t(3, 129).attention(t(3, 129), t(3, 129), heads=1)
    with pytest.raises(fg.FerrogradError, match="same device"):
        q.attention(fg.Tensor.zeros([10, 8], "hip"), k, heads=4, kv_heads=2, batch=2)


def test_norm_rotate_refusals(fg, cpu):
    t = lambda *s: cpu_tensor(fg, s)  # noqa: E731
    pos = cpu_tensor(fg, (5,), np.int32)
    x = t(5, 24)
    with pytest.raises(fg.FerrogradError, match="the cpu device has no kernel"):
        x.norm_rotate(t(8), pos, heads=3)
    for args, kw, match in [
        ((t(8), pos), dict(heads=5), "do not split into 5 heads"),
        ((t(8), pos), dict(heads=8), "must be even"),
        ((t(6), pos), dict(heads=3), "weight must be f32 of shape"),
        ((t(8), t(5)), dict(heads=3), "positions must be i32"),
        ((t(8), cpu_tensor(fg, (4,), np.int32)), dict(heads=3), "positions must be i32 of shape"),
        ((t(8), pos), dict(heads=3, eps=-1.0), "eps"),
        ((t(8), pos), dict(heads=3, base=0.0), "base"),
        ((t(8), pos), dict(heads=0), "at least 1"),
    ]:
        with pytest.raises(fg.FerrogradError, match=match):
            x.norm_rotate(*args, **kw)
    with pytest.raises(fg.FerrogradError, match="at most 512"):
        t(1, 514).norm_rotate(t(514), cpu_tensor(fg, (1,), np.int32), heads=1)


def test_dropout_refusals(fg, cpu):
    x = cpu_tensor(fg, (5, 4))
    with pytest.raises(fg.FerrogradError, match="the cpu device has no kernel"):
        x.dropout(0.5, 1)
    for p in (-0.1, 1.0, float("nan")):
        with pytest.raises(fg.FerrogradError, match="p must be in"):
            x.dropout(p, 1)
    for seed, offset in ((-1, 0), (1 << 64, 0), (0, -1)):
        with pytest.raises(fg.FerrogradError, match="must be in"):
            x.dropout(0.5, seed, offset)
    with pytest.raises(fg.FerrogradError, match="must be f32"):
        cpu_tensor(fg, (5, 4), np.int32).dropout(0.5, 1)


def classes(fg, roots):
    return [it["class"] for it in fg.debug_plan(roots, fuse=True, render_hip=True)["items"]]


@pytest.mark.gpu
def test_a_projection_feeds_a_call_in_one_kernel_and_its_gradient_arrives_uncopied(fg, hip):
    # Linear's bias stays in its product's kernel, the call reads that buffer,
    # and the gradient seed g * 1 is g itself.
    layer, x = fg.Linear(64, 64, "hip"), fg.Tensor.ones([128, 64], "hip")
    g = fg.Tensor.ones([128, 64], "hip")
    y = layer(x).dropout(0.5, 1, 2)
    got = classes(fg, [y])
    assert len(got) == 2 and got[0].startswith("gemm") and got[1] == "dropout"
    q = fg.Tensor.ones([128, 64], "hip").with_requires_grad(True)
    y = q.attention(q, q, heads=2, batch=4)
    grads = y.mul(g).sum([0, 1]).gradient([q])
    assert [c for c in classes(fg, [y, grads[0]]) if c not in ("storage", "attention", "attention_grad")] == \
        ["elementwise"]  # dq + dk + dv


def test_a_call_takes_views_reshapes_literals_and_values_other_roots_share(fg):
    x = fg.Tensor.zeros([6, 8], "hip").with_requires_grad(True)
    t = x.permute([1, 0])
    assert classes(fg, [t.dropout(0.5, 1)])[-1] == "dropout"
    h = x.add(x)
    assert classes(fg, [h, h.dropout(0.5, 1)])[-1] == "dropout"
    assert classes(fg, [x.narrow(0, 2, 3).dropout(0.5, 1)])[-1] == "dropout"
    ones = x.dropout(0.5, 1).sum([0, 1]).gradient([x])  # its gradient seed is a literal 1
    assert classes(fg, ones)[-1] == "dropout"


# ── values (GPU) ────────────────────────────────────────────────────────────


def new(fg, x, grad=False):
    t = fg.Tensor.new(x, list(x.shape), "hip")
    return t.with_requires_grad(True) if grad else t


def check(name, got, want, bound):
    off = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all(), name
    worst = np.max(off / bound)
    assert worst <= 1.0, (name, worst, np.unravel_index(np.argmax(off / bound), off.shape))


def run_attention(fg, q, k, v, g, **kw):
    kw = dict(kw)
    if kw.get("lengths") is not None:
        kw["lengths"] = new(fg, np.asarray(kw["lengths"], np.int32))
    tq, tk, tv = new(fg, q, True), new(fg, k, True), new(fg, v, True)
    y = tq.attention(tk, tv, **kw)
    out = {"y": y}
    if g is not None:
        grads = y.mul(new(fg, g)).sum([0, 1]).gradient([tq, tk, tv])
        out.update(zip(("dq", "dk", "dv"), grads))
    fg.Tensor.realize_many(list(out.values()))
    return {n: t.numpy() for n, t in out.items()}


def attention_inputs(seed, batch, sq, sk, heads, kv_heads, dim, spread=2.0):
    r = seeded(seed)
    f = lambda n, c, s=1.0: (s * r.standard_normal((n, c))).astype(np.float32)  # noqa: E731
    return (f(batch * sq, heads * dim, spread), f(batch * sk, kv_heads * dim), f(batch * sk, kv_heads * dim),
            f(batch * sq, heads * dim))


SHAPES = [  # batch, sq, sk, heads, kv_heads, dim, causal, lengths
    (1, 1, 1, 1, 1, 1, False, None),
    (1, 1, 1, 2, 1, 64, True, None),
    (2, 1, 300, 8, 2, 128, False, [300, 17]),
    (2, 1, 70, 5, 1, 40, False, [0, 70]),
    (3, 2, 129, 6, 3, 33, True, [129, 5, 0]),
    (1, 33, 33, 4, 4, 32, True, None),
    (2, 64, 64, 2, 2, 16, False, None),
    (2, 65, 130, 4, 1, 80, True, [130, 64]),
    (2, 130, 65, 2, 2, 72, True, None),  # the first 65 queries see nothing
    (1, 200, 31, 3, 3, 127, False, None),
    (2, 160, 160, 4, 2, 128, True, [160, 97]),
    (1, 257, 513, 2, 1, 96, False, None),
    (5, 31, 32, 5, 5, 8, True, [32, 1, 31, 2, 33]),
    (1, 1000, 1000, 1, 1, 64, True, None),
    (1, 40, 2500, 2, 2, 64, False, None),
    (2, 3, 700, 10, 2, 100, True, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(str(x) for x in s[:6]))
def test_attention_and_its_gradients(fg, hip, shape):
    batch, sq, sk, heads, kv_heads, dim, causal, lengths = shape
    q, k, v, g = attention_inputs(3, batch, sq, sk, heads, kv_heads, dim)
    lengths = None if lengths is None else np.asarray(lengths, np.int32)
    kw = dict(batch=batch, heads=heads, kv_heads=kv_heads, causal=causal, lengths=lengths)
    want = attention_ref.attention(q, k, v, g=g, **kw)
    got = run_attention(fg, q, k, v, g, **kw)
    for name in ("y", "dq", "dk", "dv"):
        check(name, got[name], *want[name])
    y = run_attention(fg, q, k, v, None, **kw)["y"]
    assert np.array_equal(y, got["y"])  # the same without the gradients


# Calls large enough for their forward pass to cut its operands, and of more
# workgroups than one launch of both gradients takes.
LARGE_SHAPES = [
    (17, 130, 130, 32, 16, 32, True, None),
    (8, 200, 260, 16, 8, 50, True, [260, 0, 1, 32, 33, 128, 129, 255]),
    (4, 300, 300, 16, 16, 80, False, [300, 299, 96, 7]),
    (4, 300, 270, 16, 4, 128, True, None),  # the first 30 queries see nothing
    (4, 130, 257, 32, 32, 127, False, None),
    (1, 64, 5000, 16, 16, 64, False, None),
    (1, 256, 4000, 16, 16, 64, False, None),  # keys of a query tile in parts
    (1, 520, 300, 64, 1, 64, True, [290]),  # queries of a key tile in parts
    (1, 600, 600, 24, 24, 100, True, None),
    (16, 130, 130, 20, 20, 64, True, [130 - 8 * i for i in range(16)]),
    (16, 130, 130, 20, 10, 96, False, None),
    (16, 130, 260, 20, 10, 120, True, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", LARGE_SHAPES, ids=lambda s: "x".join(str(x) for x in s[:6]))
def test_larger_attention_and_its_gradients(fg, hip, shape):
    batch, sq, sk, heads, kv_heads, dim, causal, lengths = shape
    q, k, v, g = attention_inputs(4, batch, sq, sk, heads, kv_heads, dim)
    lengths = None if lengths is None else np.asarray(lengths, np.int32)
    kw = dict(batch=batch, heads=heads, kv_heads=kv_heads, causal=causal, lengths=lengths)
    want = attention_ref.attention(q, k, v, g=g, **kw)
    got = run_attention(fg, q, k, v, g, **kw)
    for name in ("y", "dq", "dk", "dv"):
        check(name, got[name], *want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [63, 64, 65, 130])
def test_attention_of_many_short_sequences(fg, hip, batch):
    q, k, v, g = attention_inputs(15, batch, 5, 300, 2, 1, 16)
    lengths = seeded(batch).integers(0, 301, batch).astype(np.int32)
    kw = dict(batch=batch, heads=2, kv_heads=1, lengths=lengths)
    want = attention_ref.attention(q, k, v, g=g, **kw)
    got = run_attention(fg, q, k, v, g, **kw)
    for name in ("y", "dq", "dk", "dv"):
        check(name, got[name], *want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("sq", [1, 3])
@pytest.mark.parametrize("dim", [3, 30, 128])
@pytest.mark.parametrize("lengths", [[0, 2500, 7, 1300, 0, 128, 129, 2499, 1, 0], [0] * 10, [2500] * 10, [0] * 9 + [2500],
                                     [64, 0, 0, 0, 0, 0, 0, 0, 0, 0]], ids=["mixed", "none", "all", "last", "first"])
def test_tokens_of_sequences_of_unlike_lengths(fg, hip, lengths, dim, sq):
    q, k, v, _ = attention_inputs(16, 10, sq, 2500, 12, 6, dim)
    lengths = np.asarray(lengths, np.int32)
    kw = dict(batch=10, heads=12, kv_heads=6, causal=sq > 1, lengths=lengths)
    want = attention_ref.attention(q, k, v, **kw)
    check("y", run_attention(fg, q, k, v, None, **kw)["y"], *want["y"])


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [1, 2, 3, 5, 6, 7, 61, 62, 66, 125, 126])
@pytest.mark.parametrize("sq,sk", [(2, 1200), (40, 45)])
def test_attention_of_heads_that_end_within_a_vector(fg, hip, sq, sk, dim):
    q, k, v, g = attention_inputs(100 + dim, 2, sq, sk, 6, 3, dim)
    kw = dict(batch=2, heads=6, kv_heads=3, causal=True, lengths=np.array([sk - 3, 31], np.int32))
    want = attention_ref.attention(q, k, v, g=g, **kw)
    got = run_attention(fg, q, k, v, g, **kw)
    for name in ("y", "dq", "dk", "dv"):
        check(name, got[name], *want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("sq", [1, 90])
def test_hidden_keys_may_hold_anything(fg, hip, sq):
    q, k, v, g = attention_inputs(5, 2, sq, 90, 4, 2, 48)
    kw = dict(batch=2, heads=4, kv_heads=2, causal=sq > 1, lengths=np.array([50, 0], np.int32))
    clean = run_attention(fg, q, k, v, g, **kw)
    junk = np.array([np.nan, np.inf, -np.inf, np.finfo(np.float32).max, np.finfo(np.float32).min], np.float32)
    for x in (k, v):
        x[50:90] = junk[np.arange(40 * x.shape[1]) % 5].reshape(40, -1)
        x[90:] = junk[np.arange(90 * x.shape[1]) % 5].reshape(90, -1)
    dirty = run_attention(fg, q, k, v, g, **kw)
    for n in clean:
        assert np.array_equal(clean[n], dirty[n]), n
    assert not dirty["y"][sq:].any() and not dirty["dk"][50:].any() and not dirty["dv"][50:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-18, 1e-6, 1e6, 1e15])
def test_attention_of_small_and_large_values(fg, hip, size):
    # The scores stay of a few units: q shrinks as k grows.
    q, k, v, g = attention_inputs(6, 1, 100, 100, 2, 2, 64)
    q, k, v, g = (q / np.float32(size)), (k * np.float32(size)), v * np.float32(size), g / np.float32(size)
    kw = dict(batch=1, heads=2, kv_heads=2, causal=True)
    want = attention_ref.attention(q, k, v, g=g, **kw)
    got = run_attention(fg, q, k, v, g, **kw)
    for name in want:
        check(name, got[name], *want[name])


@pytest.mark.gpu
def test_attention_with_sharp_rows_and_values_of_unlike_sizes(fg, hip):
    # Scores of hundreds (one key takes the row), values whose blocks of rows
    # differ by 2^40, a zero block, and a scale of its own.
    q, k, v, g = attention_inputs(7, 1, 150, 300, 4, 1, 64, spread=40.0)
    v *= (2.0 ** np.linspace(-20, 20, 300))[:, None].astype(np.float32)
    v[64:128] = 0
    g *= (2.0 ** np.linspace(10, -10, 150))[:, None].astype(np.float32)
    kw = dict(batch=1, heads=4, kv_heads=1, scale=0.3)
    want = attention_ref.attention(q, k, v, g=g, **kw)
    got = run_attention(fg, q, k, v, g, **kw)
    for name in want:
        check(name, got[name], *want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-18, 1e15])
def test_larger_attention_of_small_and_large_values(fg, hip, size):
    q, k, v, g = attention_inputs(12, 1, 400, 800, 32, 32, 64)
    q, k, v, g = (q / np.float32(size)), (k * np.float32(size)), v * np.float32(size), g / np.float32(size)
    kw = dict(batch=1, heads=32, kv_heads=32, causal=True)
    want = attention_ref.attention(q, k, v, g=g, **kw)
    got = run_attention(fg, q, k, v, g, **kw)
    for name in want:
        check(name, got[name], *want[name])


@pytest.mark.gpu
def test_larger_attention_with_sharp_rows_and_values_of_unlike_sizes(fg, hip):
    q, k, v, g = attention_inputs(13, 1, 400, 800, 32, 8, 64, spread=40.0)
    v *= (2.0 ** np.linspace(-20, 20, 800))[:, None].astype(np.float32)
    v[64:128] = 0
    g *= (2.0 ** np.linspace(10, -10, 400))[:, None].astype(np.float32)
    kw = dict(batch=1, heads=32, kv_heads=8, scale=0.3)
    want = attention_ref.attention(q, k, v, g=g, **kw)
    got = run_attention(fg, q, k, v, g, **kw)
    for name in want:
        check(name, got[name], *want[name])


@pytest.mark.gpu
def test_larger_attention_with_anything_behind_the_lengths(fg, hip):
    q, k, v, g = attention_inputs(14, 2, 300, 700, 32, 16, 64)
    kw = dict(batch=2, heads=32, kv_heads=16, lengths=np.array([500, 3], np.int32))
    clean = run_attention(fg, q, k, v, g, **kw)
    junk = np.array([np.nan, np.inf, -np.inf, np.finfo(np.float32).max, np.finfo(np.float32).min], np.float32)
    for x in (k, v):
        for rows in (slice(500, 700), slice(703, 1400)):
            x[rows] = junk[np.arange(x[rows].size) % 5].reshape(x[rows].shape)
    dirty = run_attention(fg, q, k, v, g, **kw)
    for n in clean:
        assert np.array_equal(clean[n], dirty[n]), n
    for n in ("dk", "dv"):
        assert not dirty[n][500:700].any() and not dirty[n][703:].any()


@pytest.mark.gpu
def test_attention_of_one_tensor_with_itself(fg, hip):
    x = seeded(8).standard_normal((70, 64)).astype(np.float32)
    g = seeded(9).standard_normal((70, 64)).astype(np.float32)
    t = new(fg, x, True)
    d = t.attention(t, t, heads=2, causal=True).mul(new(fg, g)).sum([0, 1]).gradient([t])[0].numpy()
    want = attention_ref.attention(x, x, x, 1, 2, 2, causal=True, g=g)
    check("dx", d, sum(want[n][0] for n in ("dq", "dk", "dv")), 2 * sum(want[n][1] for n in ("dq", "dk", "dv")))


def directional(f, xs, ds, h=1e-5):
    return (f(*[x + h * d for x, d in zip(xs, ds)]) - f(*[x - h * d for x, d in zip(xs, ds)])) / (2 * h)


@pytest.mark.gpu
def test_attention_gradients_against_differences(fg, hip):
    batch, sq, sk, heads, kv_heads, dim = 2, 37, 50, 4, 2, 24
    q, k, v, g = attention_inputs(10, batch, sq, sk, heads, kv_heads, dim)
    kw = dict(batch=batch, heads=heads, kv_heads=kv_heads, causal=True, lengths=np.array([50, 33], np.int32))
    got = run_attention(fg, q, k, v, g, **kw)
    r = seeded(11)
    ds = [r.standard_normal(x.shape) for x in (q, k, v)]
    f = lambda *xs: float((attention_ref.attention(*xs, **kw)["y"][0] * g).sum())  # noqa: E731
    want = directional(f, [x.astype(np.float64) for x in (q, k, v)], ds)
    terms = [np.abs(got[n] * d).sum() for n, d in zip(("dq", "dk", "dv"), ds)]
    have = sum(float((got[n].astype(np.float64) * d).sum()) for n, d in zip(("dq", "dk", "dv"), ds))
    # The difference is good to h^2 (1e-10) of third derivatives and 2^-53 / h (1e-11) of the sum's terms.
    assert abs(have - want) <= 1e-5 * sum(terms)


def norm_rotate_ref(x, w, pos, heads, eps, base, g=None):
    """(value, bound) of y, dx, dweight in float64."""
    n, d = x.shape[0], x.shape[1] // heads
    x, w = x.astype(np.float64).reshape(n, heads, d), w.astype(np.float64)
    a = pos.astype(np.float64)[:, None] * base ** (-np.arange(d // 2) * 2.0 / d)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    rot = lambda z, s: np.concatenate([z[..., :d // 2] * c - z[..., d // 2:] * s,  # noqa: E731
                                       z[..., d // 2:] * c + z[..., :d // 2] * s], 2)
    swap = lambda z: np.concatenate([z[..., d // 2:], z[..., :d // 2]], 2)  # noqa: E731
    eps = float(np.float32(eps))
    r = ((x * x).mean(2, keepdims=True) + eps) ** -0.5
    nx = x * r
    z = nx * w
    y = rot(z, s)
    # r: d products and sums, a root and a quotient; the angle's cosine and
    # sine to 8 half steps of 1; three more roundings and the pair's sum.
    k = (d + 24) * U
    pair = np.abs(z) + swap(np.abs(z))
    out = {"y": (y.reshape(n, -1), (k * pair).reshape(n, -1) + 1e-38)}
    if g is None:
        return out
    g = g.astype(np.float64).reshape(n, heads, d)
    gr = rot(g, -s)
    gm = np.abs(g) + swap(np.abs(g))
    gw = gr * w
    mean = (gw * nx).mean(2, keepdims=True)
    dx = r * (gw - nx * mean)
    dxb = 2 * k * r * (gm * np.abs(w) + np.abs(nx) * (gm * np.abs(w) * np.abs(nx)).mean(2, keepdims=True))
    out["dx"] = dx.reshape(n, -1), dxb.reshape(n, -1) + 1e-38
    # Sums over all rows, in runs of registers and trees: at most the number of
    # rows in order.
    out["dweight"] = (gr * nx).sum((0, 1)), (2 * k + n * heads * U) * (gm * np.abs(nx)).sum((0, 1)) + 1e-38
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,dim,far", [(1, 1, 2, 1), (1, 3, 6, 9), (7, 5, 64, 1 << 20), (33, 2, 74, 33),
                                                  (5, 1, 8, 100), (300, 7, 128, 4096), (2, 40, 512, 2), (3, 2, 300, 50),
                                                  (4, 3, 510, 1 << 30), (3000, 8, 96, 5000), (20000, 3, 20, 20000),
                                                  (2, 2, 260, 7), (3, 1, 30, 10), (9, 2, 12, 10)])
def test_norm_rotate_and_its_gradients(fg, hip, tokens, heads, dim, far):
    r = seeded(dim)
    x = (3 * r.standard_normal((tokens, heads * dim))).astype(np.float32)
    w = (1 + 0.3 * r.standard_normal(dim)).astype(np.float32)
    g = r.standard_normal(x.shape).astype(np.float32)
    pos = r.integers(-far, far, tokens).astype(np.int32)
    pos[0] = far - 1
    want = norm_rotate_ref(x, w, pos, heads, 1e-5, 500000.0, g)
    tx, tw = new(fg, x, True), new(fg, w, True)
    y = tx.norm_rotate(tw, new(fg, pos), heads, eps=1e-5, base=500000.0)
    dx, dw = y.mul(new(fg, g)).sum([0, 1]).gradient([tx, tw])
    fg.Tensor.realize_many([y, dx, dw])
    for name, t in (("y", y), ("dx", dx), ("dweight", dw)):
        check(name, t.numpy(), *want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [4, 10, 14, 66, 130, 250, 258, 386])
def test_norm_rotate_of_halves_that_end_within_a_vector(fg, hip, dim):
    r = seeded(1000 + dim)
    tokens, heads = 37, 3
    x = (3 * r.standard_normal((tokens, heads * dim))).astype(np.float32)
    w = (1 + 0.3 * r.standard_normal(dim)).astype(np.float32)
    g = r.standard_normal(x.shape).astype(np.float32)
    pos = r.integers(0, 4096, tokens).astype(np.int32)
    want = norm_rotate_ref(x, w, pos, heads, 1e-6, 10000.0, g)
    tx, tw = new(fg, x, True), new(fg, w, True)
    y = tx.norm_rotate(tw, new(fg, pos), heads)
    dx, dw = y.mul(new(fg, g)).sum([0, 1]).gradient([tx, tw])
    fg.Tensor.realize_many([y, dx, dw])
    for name, t in (("y", y), ("dx", dx), ("dweight", dw)):
        check(name, t.numpy(), *want[name])


@pytest.mark.gpu
def test_norm_rotate_of_zero_rows_and_gradients_against_differences(fg, hip):
    r = seeded(2)
    x = r.standard_normal((6, 32)).astype(np.float32)
    x[2, :16] = 0  # a head of zeros: r = eps^(-1/2)
    w, g = r.standard_normal(16).astype(np.float32), r.standard_normal((6, 32)).astype(np.float32)
    pos = np.arange(6, dtype=np.int32)
    tx, tw = new(fg, x, True), new(fg, w, True)
    y = tx.norm_rotate(tw, new(fg, pos), 2, eps=1e-2)
    dx, dw = (t.numpy() for t in y.mul(new(fg, g)).sum([0, 1]).gradient([tx, tw]))
    assert not y.numpy()[2, :16].any()
    ds = [r.standard_normal(x.shape), r.standard_normal(w.shape)]

    def f(a, b):
        n = a.reshape(6, 2, 16)
        z = n / np.sqrt((n * n).mean(2, keepdims=True) + float(np.float32(1e-2))) * b
        t = pos[:, None] * 10000.0 ** (-np.arange(8) / 8.0)
        c, s = np.cos(t)[:, None], np.sin(t)[:, None]
        return float((np.concatenate([z[..., :8] * c - z[..., 8:] * s, z[..., 8:] * c + z[..., :8] * s], 2).reshape(6, 32) * g).sum())

    want = directional(f, [x.astype(np.float64), w.astype(np.float64)], ds, 1e-6)
    have = sum(float((t.astype(np.float64) * d).sum()) for t, d in zip((dx, dw), ds))
    assert abs(have - want) <= 1e-5 * sum(np.abs(t * d).sum() for t, d in zip((dx, dw), ds))


def philox(n, seed, offset):
    """The words of Philox4x32-10, from its definition."""
    m = np.uint64(0xFFFFFFFF)
    at = np.arange((n + 3) // 4, dtype=np.uint64)
    c = [at & m, at >> np.uint64(32), np.full_like(at, offset & 0xFFFFFFFF), np.full_like(at, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[:n]


def test_philox_known_words():
    # The generator's published test vectors: all zeros, all ones, digits of pi.
    assert [hex(w) for w in philox(4, 0, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


def dropped(x, p, seed, offset):
    keep = philox(x.size, seed, offset).reshape(x.shape) >= int(p * 2 ** 32)
    return np.where(keep, x * np.float32(1.0 / (1.0 - p)), np.float32(0))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,p,seed,offset", [((1,), 0.5, 0, 0), ((3,), 0.9, 1, 2), ((5, 1), 1e-3, 1 << 63, 0),
                                                 ((256, 128), 0.5, 42, 1), ((1001, 77), 0.1, (1 << 64) - 1, (1 << 64) - 1),
                                                 ((2, 3, 5, 7), 0.25, 7, 1 << 32), ((9, 9), 0.0, 3, 3),
                                                 ((1 << 20,), 0.999999, 5, 6)])
def test_dropout_and_its_gradient(fg, hip, shape, p, seed, offset):
    r = seeded(1)
    x, g = r.standard_normal(shape).astype(np.float32), r.standard_normal(shape).astype(np.float32)
    t = new(fg, x, True)
    y = t.dropout(p, seed, offset)
    dx = y.mul(new(fg, g)).sum(list(range(len(shape)))).gradient([t])[0]
    fg.Tensor.realize_many([y, dx])
    # One rounded product a kept element: the same bits.
    assert np.array_equal(y.numpy(), dropped(x, p, seed, offset))
    assert np.array_equal(dx.numpy(), dropped(g, p, seed, offset))


@pytest.mark.gpu
def test_dropped_elements_are_zero_whatever_they_held(fg, hip):
    x = np.full(1000, np.nan, np.float32)
    x[::2] = np.inf
    y = new(fg, x).dropout(0.5, 9).numpy()
    keep = philox(1000, 9, 0) >= 1 << 31
    assert not y[~keep].any() and not np.isfinite(y[keep]).any()


# ── calls in sequences (GPU) ────────────────────────────────────────────────


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_replayed_calls_take_their_seeds_from_the_call(fg, hip, graphs):
    import contextlib

    x = seeded(4).standard_normal((40, 50)).astype(np.float32)
    t = new(fg, x)
    fg.clear_caches()
    with graphs_on(fg) if graphs else contextlib.nullcontext():
        for step in range(6):
            h0 = fg.plan_stats()["hits"]
            # Two calls in one plan: the second's offset passes values the first's had.
            y = t.dropout(0.5, 77, 3 + step).mul(t).dropout(0.3, 78, 4 + 2 * step).realize()
            want = dropped(dropped(x, 0.5, 77, 3 + step) * x, 0.3, 78, 4 + 2 * step)
            assert np.array_equal(y.numpy(), want), step
            assert step == 0 or fg.plan_stats()["hits"] > h0
    # Equal words share one node: a plan of its own, never another call's.
    y = t.dropout(0.5, 5, 5).dropout(0.5, 5, 5).numpy()
    assert np.array_equal(y, dropped(dropped(x, 0.5, 5, 5), 0.5, 5, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_replayed_attention_with_its_gradients_reads_the_new_inputs(fg, hip, graphs):
    import contextlib

    with graphs_on(fg) if graphs else contextlib.nullcontext():
        for step in range(5):
            q, k, v, g = attention_inputs(20 + step, 2, 70, 70, 4, 2, 64)
            kw = dict(batch=2, heads=4, kv_heads=2, causal=True, lengths=np.array([70, 20 + step], np.int32))
            got = run_attention(fg, q, k, v, g, **kw)
            want = attention_ref.attention(q, k, v, g=g, **kw)
            for name in want:
                check((step, name), got[name], *want[name])
            # A larger call in between takes a larger workspace.
            big = attention_inputs(30, 1, 300 + 50 * step, 300 + 50 * step, 2, 2, 64)
            run_attention(fg, *big, batch=1, heads=2)


@pytest.mark.gpu
def test_gradients_realised_after_their_loss(fg, hip):
    # The forward call runs first and alone; the gradients then read the
    # outputs and sums it left.
    q, k, v, g = attention_inputs(12, 1, 60, 60, 2, 2, 32)
    tq, tk, tv = (new(fg, x, True) for x in (q, k, v))
    y = tq.attention(tk, tv, heads=2, causal=True)
    loss = y.mul(new(fg, g)).sum([0, 1])
    loss.backward()
    loss.realize()
    want = attention_ref.attention(q, k, v, 1, 2, 2, causal=True, g=g)
    for name, t in (("dq", tq), ("dv", tv), ("dk", tk)):  # one at a time
        check(name, t.grad().numpy(), *want[name])


@pytest.mark.gpu
def test_gradients_of_gradients(fg, hip):
    # Dropout's is its own again; the others' are refused.
    x = seeded(30).standard_normal((12, 16)).astype(np.float32)
    t = new(fg, x, True)
    g = t.dropout(0.5, 3).mul(t).sum([0, 1]).gradient([t])[0]  # 2 m x, m the mask times 2
    d = g.mul(g).sum([0, 1]).gradient([t])[0].numpy()
    m = dropped(np.ones_like(x), 0.5, 3, 0)
    assert np.array_equal(d, 8 * m * m * x)  # all powers of two but x
    w, pos = new(fg, np.ones(8, np.float32), True), new(fg, np.arange(12, dtype=np.int32))
    for y in (t.attention(t, t, heads=2), t.norm_rotate(w, pos, heads=2)):
        g = y.sum([0, 1]).gradient([t])[0]
        with pytest.raises(fg.FerrogradError, match="gradient not implemented"):
            g.mul(g).sum([0, 1]).gradient([t])


@pytest.mark.gpu
def test_calls_read_views_and_literals_and_update_in_place(fg, hip):
    r = seeded(40)
    x, m = r.standard_normal((12, 8)).astype(np.float32), r.standard_normal((8, 12)).astype(np.float32)
    t, tm = new(fg, x, True), new(fg, m)
    assert np.array_equal(t.permute([1, 0]).dropout(0.5, 1).numpy(), dropped(x.T, 0.5, 1, 0))
    assert np.array_equal(t.narrow(0, 5, 6).dropout(0.5, 1).numpy(), dropped(x[5:11], 0.5, 1, 0))
    assert np.array_equal(t.narrow(1, 3, 4).dropout(0.5, 1).numpy(), dropped(x[:, 3:7], 0.5, 1, 0))
    # Read by the call and by another root: both see the same values.
    h = t.permute([1, 0]).add(tm)
    y = h.dropout(0.5, 2)
    fg.Tensor.realize_many([h, y])
    assert np.array_equal(h.numpy(), x.T + m) and np.array_equal(y.numpy(), dropped(x.T + m, 0.5, 2, 0))
    # A gradient that is a literal, and one that sums over a broadcast.
    ones = t.dropout(0.5, 3).sum([0, 1]).gradient([t])[0].numpy()
    assert np.array_equal(ones, dropped(np.ones_like(x), 0.5, 3, 0))
    row = new(fg, x[:1], True)
    d = row.expand([12, 8]).dropout(0.5, 4).sum([0, 1]).gradient([row])[0].numpy()
    assert np.array_equal(d, dropped(np.ones_like(x), 0.5, 4, 0).sum(0, keepdims=True))
    # Attention over transposed, narrowed keys.
    kv = r.standard_normal((16, 20)).astype(np.float32)
    tkv = new(fg, kv)
    k, v = tkv.narrow(0, 0, 8).permute([1, 0]), tkv.narrow(0, 8, 8).permute([1, 0])
    check("y", t.attention(k, v, heads=2).numpy(), *attention_ref.attention(x, kv[:8].T, kv[8:].T, 1, 2, 2)["y"])
    # In place: the call reads what the store replaces.
    z = new(fg, x)
    for step in range(3):
        z.assign(z.dropout(0.5, 5, step))
        z.realize()
    assert np.array_equal(z.numpy(), dropped(dropped(dropped(x, 0.5, 5, 0), 0.5, 5, 1), 0.5, 5, 2))


@pytest.mark.gpu
def test_two_calls_of_one_realisation_share_the_workspace(fg, hip):
    q, k, v, _ = attention_inputs(41, 1, 300, 300, 4, 4, 64)
    tq, tk, tv = (new(fg, x) for x in (q, k, v))
    want = attention_ref.attention(q, k, v, 1, 4, 4)["y"]
    for step in range(3):
        small = tq.attention(tk, tv, heads=4)
        big = tq.attention(tk.permute([1, 0]).permute([1, 0]).contiguous(), tv, heads=4, causal=True)
        fg.Tensor.realize_many([small, big])
        check("small", small.numpy(), *want)
        check("big", big.numpy(), *attention_ref.attention(q, k, v, 1, 4, 4, causal=True)["y"])
        fg.clear_caches() if step == 1 else None


@pytest.mark.gpu
def test_the_same_inputs_give_the_same_bits(fg, hip):
    q, k, v, g = attention_inputs(13, 2, 300, 300, 4, 2, 64)
    kw = dict(batch=2, heads=4, kv_heads=2, causal=True)
    a, b = run_attention(fg, q, k, v, g, **kw), run_attention(fg, q, k, v, g, **kw)
    for n in a:
        assert np.array_equal(a[n], b[n]), n


# ── together, as layers ─────────────────────────────────────────────────────


def test_layers_refuse_what_their_calls_would(fg, cpu):
    from ferrograd_amd.attention import SelfAttention
    from ferrograd_amd.mlp import Mlp, train_steps_native

    for kw, match in [(dict(heads=5), "do not split"), (dict(heads=32), "must be even"),
                      (dict(heads=4, kv_heads=3), "do not share"), (dict(heads=1, head_dim=130), "at most 128")]:
        with pytest.raises(fg.FerrogradError, match=match):
            SelfAttention(32, device=cpu, **kw)
    with pytest.raises(fg.FerrogradError, match="p must be in"):
        fg.Dropout(1.0)
    model = Mlp((4, 3, 2), cpu, dropout=0.5)
    with pytest.raises(fg.FerrogradError, match="run no dropout"):
        train_steps_native(model, None, None, None, 1)
    x = cpu_tensor(fg, (5, 4))
    assert model.train(False).forward(x).shape == (5, 2)  # and without dropout any device does


class Torch64:
    """The layers in float64 on the CPU."""

    @staticmethod
    def norm_rotate(x, w, pos, heads, eps, base):
        import torch

        n, d = x.shape[0], x.shape[1] // heads
        z = x.reshape(n, heads, d)
        z = z / torch.sqrt((z * z).mean(2, keepdim=True) + eps) * w
        a = pos[:, None].double() * base ** (-torch.arange(d // 2).double() * 2 / d)
        c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
        l, r = z[..., :d // 2], z[..., d // 2:]
        return torch.cat([l * c - r * s, r * c + l * s], 2).reshape(n, -1)

    @staticmethod
    def attention(q, k, v, heads, kv_heads, batch, lengths):
        import torch

        split = lambda t, h: t.reshape(batch, -1, h, t.shape[1] // h).transpose(1, 2)  # noqa: E731
        q, k, v = split(q, heads), *(split(t, kv_heads).repeat_interleave(heads // kv_heads, 1) for t in (k, v))
        s = q @ k.transpose(2, 3) / q.shape[3] ** 0.5
        n = s.shape[2]
        hide = torch.ones(n, n, dtype=torch.bool).triu(1)[None, None] | (
            torch.arange(n)[None, None, None] >= lengths[:, None, None, None])
        y = torch.softmax(s.masked_fill(hide, float("-inf")), 3) @ v
        return y.transpose(1, 2).reshape(batch * n, -1)


@pytest.mark.gpu
def test_a_self_attention_layer_and_its_gradients(fg, hip):
    import torch

    from ferrograd_amd.attention import SelfAttention

    batch, n, features, heads, kv_heads = 3, 41, 48, 6, 2
    fg.reset_init_seed(3)
    layer = SelfAttention(features, heads, kv_heads, head_dim=16, device=hip, dropout=0.25, seed=9)
    r = seeded(31)
    x, g = (r.standard_normal((batch * n, features)).astype(np.float32) for _ in range(2))
    pos = np.tile(np.arange(n, dtype=np.int32), batch)
    lengths = np.array([41, 7, 30], np.int32)
    tx, tp, tl, tg = new(fg, x, True), new(fg, pos), new(fg, lengths), new(fg, g)
    for step in range(3):  # the plan of the first step, then its replays, each with the next mask
        y = layer(tx, tp, batch, tl)
        params = layer.parameters()
        grads = y.mul(tg).sum([0, 1]).gradient([tx, *params])
        fg.Tensor.realize_many([y, *grads])
        ps = [torch.tensor(p.numpy().astype(np.float64), requires_grad=True) for p in (tx, *params)]
        px, wq, wk, wv, wo, nq, nk = ps
        q = Torch64.norm_rotate(px @ wq.T, nq, torch.tensor(pos), heads, 1e-6, 10000.0)
        k = Torch64.norm_rotate(px @ wk.T, nk, torch.tensor(pos), kv_heads, 1e-6, 10000.0)
        out = Torch64.attention(q, k, px @ wv.T, heads, kv_heads, batch, torch.tensor(lengths)) @ wo.T
        keep = philox(out.numel(), 9, step).reshape(out.shape) >= 1 << 30
        want = out * torch.tensor(keep / 0.75)
        want_grads = torch.autograd.grad((want * torch.tensor(g.astype(np.float64))).sum(), ps)
        # Each of the nine products, norms and softmaxes on a value's way is off
        # by at most its terms (features, heads' sizes, keys, tokens summed over)
        # times half a step of its terms' magnitudes; 16 for magnitudes over sums.
        tol = 9 * 16 * (features + heads * 16 + n + batch * n) * U
        for name, got, ref in [("y", y, want)] + list(zip("x wq wk wv wo nq nk".split(), grads, want_grads)):
            ref = ref.detach().numpy()
            off = np.linalg.norm(got.numpy() - ref) / np.linalg.norm(ref)
            assert off <= tol, (step, name, off, tol)
    before = layer.train(False)(tx, tp, batch, tl).numpy()
    assert np.array_equal(before, layer(tx, tp, batch, tl).numpy())  # no dropout


@pytest.mark.gpu
def test_a_sequence_classifier_trains(fg, hip):
    # Two layers around a residual, a classifier on top, SGD in place: every
    # parameter moves and the loss is the one that the parameters before it give.
    from ferrograd_amd.attention import SelfAttention

    fg.reset_init_seed(5)
    layers = [SelfAttention(32, 4, 2, device=hip, dropout=0.1, seed=i) for i in range(2)]
    head = fg.Linear(32, 5, hip)
    params = [p for l in layers for p in l.parameters()] + head.parameters()
    opt = fg.Sgd(params, 0.05)
    r = seeded(32)
    pos = new(fg, np.tile(np.arange(20, dtype=np.int32), 4))
    before = [p.numpy().copy() for p in params]
    for step in range(4):
        h = new(fg, r.standard_normal((80, 32)).astype(np.float32))
        t = new(fg, np.eye(5, dtype=np.float32)[r.integers(0, 5, 80)])
        for l in layers:
            h = h.add(l(h, pos, 4))
        loss = head(h).cross_entropy(t)
        opt.zero_grad()
        loss.backward()
        opt.step()
        assert np.isfinite(loss.to_vec()[0])
    for p, b in zip(params, before):
        assert np.isfinite(p.numpy()).all() and not np.array_equal(p.numpy(), b)


@pytest.mark.gpu
def test_an_mlp_with_dropout_takes_the_masks_gradient(fg, hip):
    from ferrograd_amd.mlp import Mlp, synthetic_batch, train_step

    dims, lr = (24, 40, 33, 6), 0.5
    fg.reset_init_seed(7)
    model = Mlp(dims, hip, dropout=0.5, seed=70)
    opt = fg.Sgd(model.parameters(), lr)
    xs, ts = synthetic_batch(50, 24, 6, 1, 2)
    x, t = new(fg, xs), new(fg, ts)
    for step in range(4):
        p0 = [p.numpy().astype(np.float64) for p in model.parameters()]
        zs = []
        loss = train_step(model, opt, x, t, zs).to_vec()[0]
        hs, h = [xs.astype(np.float64)], xs.astype(np.float64)
        masks = []
        for i in range(3):
            z = h @ p0[2 * i].T + p0[2 * i + 1]
            if i < 2:
                # The device's own signs: a value within rounding of 0 may fall on either side.
                on = zs[i].numpy() > 0
                masks.append((philox(z.size, 70 + i, step).reshape(z.shape) >= 1 << 31) * 2.0 * on)
                h = z * masks[-1]
                hs.append(h)
        logp = z - z.max(1, keepdims=True)
        logp -= np.log(np.exp(logp).sum(1, keepdims=True))
        assert abs(loss + (ts * logp).sum() / 50) <= 1e-5
        dz = (np.exp(logp) - ts) / 50
        for i in reversed(range(3)):
            for j, want in ((2 * i, dz.T @ hs[i]), (2 * i + 1, dz.sum(0))):
                got = (p0[j] - model.parameters()[j].numpy()) / lr
                # The update's rounding, half a step of the parameter over lr, and 128 for the products before.
                bound = U * (np.abs(p0[j]) + 1) * 2 / lr + 128 * U * np.abs(want).max()
                assert np.abs(got - want).max() <= bound.max(), (step, j)
            if i:
                dz = (dz @ p0[2 * i]) * masks[i - 1]
