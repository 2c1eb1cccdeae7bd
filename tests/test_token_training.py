"""Embedding, layer norm, the loss of token labels and clipping to a global norm:
refusals, plans, values against float64 with bounds from their roundings,
gradients against their formulas and against differences, and a trained model of
them together."""
import numpy as np
import pytest

from conftest import graphs_on, seeded

U = 2.0 ** -24  # half a step of float32, relative
TINY = 2.0 ** -126  # below it steps no longer shrink


def cpu_tensor(fg, shape, dtype=np.float32):
    return fg.Tensor.new(np.zeros(shape, dtype), list(shape), "cpu")


def new(fg, x, grad=False):
    t = fg.Tensor.new(x, list(x.shape), "hip")
    return t.with_requires_grad(True) if grad else t


def check(name, got, want, bound):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all(), name
    worst = np.max(off / (bound + TINY))
    assert worst <= 1.0, (name, worst, np.unravel_index(np.argmax(off / (bound + TINY)), off.shape))


def normal(seed, *shape):
    return seeded(seed).standard_normal(shape).astype(np.float32)


def weighted(fg, y, g, wrt):
    """y and the gradients of sum(y * g)."""
    grads = y.mul(new(fg, g)).sum([0, 1]).gradient(wrt)
    fg.Tensor.realize_many([y] + grads)
    return [t.numpy() for t in [y] + grads]


# ── refusals and plans (no GPU) ─────────────────────────────────────────────


def test_embedding_refusals(fg, cpu):
    w, ids = cpu_tensor(fg, (5, 3)), cpu_tensor(fg, (4,), np.int32)
    with pytest.raises(fg.FerrogradError, match="the cpu device has no kernel"):
        w.embedding(ids)
    for weight, bad, kw, match in [
        (cpu_tensor(fg, (5, 3), np.int32), ids, {}, "weight must be f32"),
        (cpu_tensor(fg, (15,)), ids, {}, "weight must be 2D"),
        (cpu_tensor(fg, (0, 3)), ids, {}, "weight is empty"),
        (w, cpu_tensor(fg, (4,)), {}, "ids must be i32"),
        (w, cpu_tensor(fg, (2, 2), np.int32), {}, "ids must be i32 of one dimension"),
        (w, cpu_tensor(fg, (0,), np.int32), {}, "ids are empty"),
        (w, ids, dict(scale=float("inf")), "scale must be finite"),
        (w, ids, dict(scale=1e39), "scale must be finite"),
    ]:
        with pytest.raises(fg.FerrogradError, match=match):
            weight.embedding(bad, **kw)
    with pytest.raises(fg.FerrogradError, match="same device"):
        w.embedding(fg.Tensor.zeros([4], "hip", np.int32))
    with pytest.raises(TypeError):
        w.embedding([1, 2])
    with pytest.raises(fg.FerrogradError, match=r"must have shape \[4, 3\], got \[5, 3\]"):
        fg.Embedding(4, 3, cpu, weight=w)


def test_layer_norm_refusals(fg, cpu):
    x, w = cpu_tensor(fg, (5, 6)), cpu_tensor(fg, (6,))
    with pytest.raises(fg.FerrogradError, match="the cpu device has no kernel"):
        x.layer_norm(w, w)
    for bad, kw, match in [
        ((cpu_tensor(fg, (5,)),), {}, "weight must be f32 of shape"),
        ((cpu_tensor(fg, (6,), np.int32),), {}, "weight must be f32 of shape"),
        ((w, cpu_tensor(fg, (1, 6))), {}, "bias must be f32 of shape"),
        ((w,), dict(eps=-1.0), "eps"),
        ((w,), dict(eps=1e-46), "eps"),
        ((w,), dict(eps=float("nan")), "eps"),
        ((w,), dict(eps=1e39), "eps"),
    ]:
        with pytest.raises(fg.FerrogradError, match=match):
            x.layer_norm(*bad, **kw)
    with pytest.raises(fg.FerrogradError, match="must be 2D"):
        w.layer_norm(w)
    with pytest.raises(fg.FerrogradError, match="is empty"):
        cpu_tensor(fg, (0, 6)).layer_norm(w)
    with pytest.raises(fg.FerrogradError, match="same device"):
        x.layer_norm(w, fg.Tensor.zeros([6], "hip"))


def test_token_cross_entropy_refusals(fg, cpu):
    x, labels = cpu_tensor(fg, (5, 6)), cpu_tensor(fg, (5,), np.int32)
    with pytest.raises(fg.FerrogradError, match="the cpu device has no kernel"):
        x.token_cross_entropy(labels)
    for logits, bad, match in [
        (cpu_tensor(fg, (5,)), labels, "must be 2D"),
        (cpu_tensor(fg, (5, 0)), labels, "is empty"),
        (cpu_tensor(fg, (5, 6), np.int32), labels, "must be f32"),
        (x, cpu_tensor(fg, (6,), np.int32), "labels must be i32 of shape"),
        (x, cpu_tensor(fg, (5,)), "labels must be i32 of shape"),
        (x, cpu_tensor(fg, (5, 1), np.int32), "labels must be i32 of shape"),
        (x, fg.Tensor.zeros([5], "hip", np.int32), "same device"),
    ]:
        with pytest.raises(fg.FerrogradError, match=match):
            logits.token_cross_entropy(bad)


def test_norm_and_clip_refusals(fg, cpu):
    a, b = cpu_tensor(fg, (5, 6)), cpu_tensor(fg, (3,))
    for f in (lambda ts: fg.clip_norm(ts, 1.0), fg.global_norm):
        with pytest.raises(fg.FerrogradError, match="the cpu device has no kernel"):
            f([a, b])
        with pytest.raises(fg.FerrogradError, match="at least one tensor"):
            f([])
        with pytest.raises(fg.FerrogradError, match="tensor 1 must be f32"):
            f([a, cpu_tensor(fg, (2,), np.int32)])
        with pytest.raises(fg.FerrogradError, match="tensor 0 is empty"):
            f([cpu_tensor(fg, (0, 2)), a])
        with pytest.raises(fg.FerrogradError, match="same device"):
            f([a, fg.Tensor.zeros([2], "hip")])
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(fg.FerrogradError, match="max_norm must be finite and positive"):
            fg.clip_norm([a], bad)
    for bad in (None, 3, [a, 2.0], "ab"):
        with pytest.raises(TypeError):
            fg.clip_norm(bad, 1.0)
        with pytest.raises(TypeError):
            fg.Tensor.realize_many(bad)
        with pytest.raises(TypeError):
            a.gradient(bad)
    with pytest.raises(fg.FerrogradError, match="no handle"):
        fg.global_norm([a, fg.Tensor()])
    with pytest.raises(fg.FerrogradError, match="not realized"):
        a.add(a).data_ptr()
    p = cpu_tensor(fg, (2, 2)).with_requires_grad(True)
    with pytest.raises(fg.FerrogradError, match="clip_grad_norm requires parameter gradients"):
        fg.Sgd([p], 0.1).clip_grad_norm(1.0)


def classes(fg, roots):
    return [it["class"] for it in fg.debug_plan(roots, fuse=True, render_hip=True)["items"]]


def test_clips_that_differ_have_their_own_outputs(fg):
    a, b, c = (fg.Tensor.zeros([n, 5], "hip") for n in (3, 4, 6))
    calls = [fg.clip_norm([a, b], 1.0), fg.clip_norm([a, b], 2.0), fg.clip_norm([a, b, c], 1.0), fg.clip_norm([b, a], 1.0)]
    roots = [t for norm, clipped in calls for t in [norm] + clipped]
    outs = [it["output"] for it in fg.debug_plan(roots, fuse=True, render_hip=True)["items"]]
    assert len(set(outs)) == len(outs)
    got = classes(fg, roots)
    # [a, b] is summed once for both of its clips.
    assert got.count("square_sums") == 3 and got.count("clip") == 4
    again = fg.clip_norm([a, b], 1.0)
    assert len(classes(fg, roots + [again[0]] + again[1])) == len(got)


def test_many_tensors_go_in_calls_of_64(fg):
    ts = [fg.Tensor.zeros([1 + i], "hip") for i in range(130)]
    norm, clipped = fg.clip_norm(ts, 1.0)
    got = classes(fg, [norm] + clipped)
    assert got.count("square_sums") == 3 and got.count("clip") == 3 and got.count("storage") == 130 - 3 + 1
    assert classes(fg, [fg.global_norm(ts)]) == ["square_sums"] * 3 + ["norm_of_sums"]


# ── embedding (GPU) ─────────────────────────────────────────────────────────


def some_ids(kind, tokens, vocab, seed):
    r = seeded(seed)
    if kind == "one":
        return np.full(tokens, r.integers(vocab), np.int32)
    if kind == "none":
        return np.full(tokens, vocab, np.int32)
    ids = r.integers(0, vocab, tokens)
    if kind == "words":
        ids = np.minimum(np.exp(r.random(tokens) * np.log(vocab + 1.0)).astype(np.int64) - 1, vocab - 1)
    if kind == "outside":
        ids = np.where(r.random(tokens) < 0.4, r.choice([-1, vocab, -(2 ** 31), 2 ** 31 - 1], tokens), ids)
    return ids.astype(np.int32)


def embedding64(w, ids, g, scale):
    """Rows and the weight's gradient, each with its bound: a product is rounded once, of a scale rounded once; a sum
    of n products has n - 1 roundings of at most the terms' magnitudes."""
    vocab = w.shape[0]
    inside = (ids >= 0) & (ids < vocab)
    y = np.where(inside[:, None], w[np.where(inside, ids, 0)].astype(np.float64) * scale, 0.0)
    dw, size = np.zeros(w.shape), np.zeros(w.shape)
    np.add.at(dw, ids[inside], g[inside].astype(np.float64) * scale)
    np.add.at(size, ids[inside], np.abs(g[inside].astype(np.float64) * scale))
    n = np.bincount(ids[inside], minlength=vocab)[:, None]
    return (y, 2.01 * U * np.abs(y)), (dw, 1.01 * (n + 2) * U * size)


EMBEDDINGS = [  # tokens, vocab, dim
    (1, 1, 1), (1, 7, 5), (2, 3, 4), (63, 100, 3), (64, 2, 64), (65, 1000, 130), (257, 31, 77), (1000, 5000, 36),
    (4097, 300, 20), (5000, 70000, 12), (2049, 2048, 257), (300, 4, 1028), (9000, 3, 8),
    (12288, 900, 4), (12289, 900, 4), (16384, 900, 4), (16385, 1000, 5), (20000, 700, 6), (40000, 1500000, 3), (66000, 40, 4), (17000, 1023, 9), (17000, 1024, 8),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["uniform", "words", "one", "outside", "none"])
@pytest.mark.parametrize("shape", EMBEDDINGS, ids=lambda s: "x".join(map(str, s)))
def test_embedding_and_its_gradient(fg, hip, shape, kind):
    tokens, vocab, dim = shape
    w, g, ids = normal(1, vocab, dim), normal(2, tokens, dim), some_ids(kind, tokens, vocab, 3)
    tw = new(fg, w, True)
    y, dw = weighted(fg, tw.embedding(new(fg, ids), scale=dim ** 0.5), g, [tw])
    want_y, want_dw = embedding64(w, ids, g, dim ** 0.5)
    check("y", y, *want_y)
    check("dw", dw, *want_dw)
    inside = (ids >= 0) & (ids < vocab)
    assert not y[~inside].any() and not dw[np.setdiff1d(np.arange(vocab), ids[inside])].any()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,vocab,dim", [(1048577, 1000, 1), (4300001, 1000, 1), (8400000, 1500, 1), (8400000, 70000, 4)])
def test_embedding_gradient_of_millions_of_tokens(fg, hip, tokens, vocab, dim):
    # More than 256 tiles of 4096 tokens: some share a workgroup.
    ids, g = some_ids("words", tokens, vocab + 50, 5), normal(6, tokens, dim)
    w = fg.Tensor.zeros([vocab, dim], "hip").with_requires_grad(True)
    dw = w.embedding(new(fg, ids)).mul(new(fg, g)).sum([0, 1]).gradient([w])[0].numpy()
    inside = ids < vocab
    n = np.bincount(ids[inside], minlength=vocab)
    for c in range(dim):
        col = g[inside, c].astype(np.float64)
        want, size = (np.bincount(ids[inside], weights=x, minlength=vocab) for x in (col, np.abs(col)))
        check("dw", dw[:, c], want, 1.01 * (n + 2) * U * size)


@pytest.mark.gpu
def test_embedding_rows_may_hold_anything(fg, hip):
    # A row that no token reads, and gradients of ids that are no tokens, never matter.
    w, g = normal(4, 9, 6), normal(5, 8, 6)
    w[3], g[2], g[5] = np.nan, np.inf, np.nan
    ids = np.array([1, 1, -1, 8, 0, 9, 1, 2], np.int32)
    tw = new(fg, w, True)
    y, dw = weighted(fg, tw.embedding(new(fg, ids)), g, [tw])
    assert np.isfinite(y).all() and np.isfinite(dw).all()
    # One that is read does, in its own row alone.
    g[6, 1] = np.nan
    y, dw = weighted(fg, tw.embedding(new(fg, ids)), g, [tw])
    assert np.array_equal(np.argwhere(np.isnan(dw)), [[1, 1]])


# ── layer norm (GPU) ────────────────────────────────────────────────────────


def layer_norm64(x, w, b, g, eps):
    """y, dx, dw and db, each with its bound. A row's sum has no number that goes through more than `deep` additions: a
    row is spread over 16 lanes or more where it is long, then summed over them."""
    x, w, g = x.astype(np.float64), w.astype(np.float64), g.astype(np.float64)
    rows, dim = x.shape
    deep = dim / 16 + 16
    m = x.mean(1, keepdims=True)
    em = (deep + 1) * U * np.abs(x).mean(1, keepdims=True)
    c = x - m
    ec = em + U * np.abs(c)
    v = (c * c).mean(1, keepdims=True)
    # The derivative by the mean is 0; each square and the sum are rounded.
    ev = em * em + (deep + 4) * U * v
    r = 1 / np.sqrt(v + eps)
    er = r * (0.5 * ev / (v + eps) + 4 * U)
    h = c * r
    eh = ec * r + np.abs(c) * er + 2 * U * np.abs(h)
    y = h * w + (0 if b is None else b.astype(np.float64))
    ey = np.abs(w) * eh + 2 * U * (np.abs(h * w) + np.abs(y))
    u = g * w
    mu, mh = u.mean(1, keepdims=True), (u * h).mean(1, keepdims=True)
    emu = (deep + 2) * U * np.abs(u).mean(1, keepdims=True)
    emh = (deep + 3) * U * np.abs(u * h).mean(1, keepdims=True) + (np.abs(u) * eh).mean(1, keepdims=True)
    inner = u - mu - h * mh
    ei = U * np.abs(u) + emu + np.abs(h) * emh + np.abs(mh) * eh + 4 * U * (np.abs(u) + np.abs(mu) + np.abs(h * mh))
    dx, edx = r * inner, r * ei + np.abs(inner) * er + U * np.abs(r * inner)
    dw, edw = (g * h).sum(0), (np.abs(g) * eh).sum(0) + (rows + 2) * U * np.abs(g * h).sum(0)
    db, edb = g.sum(0), rows * U * np.abs(g).sum(0)
    # First-order bounds; what they leave out is far below a tenth of them.
    return [(a, 1.1 * e) for a, e in ((y, ey), (dx, edx), (dw, edw), (db, edb))]


LAYER_NORMS = [  # rows, dim
    (1, 1), (3, 2), (5, 3), (1, 4), (7, 5), (2, 31), (33, 32), (9, 33), (4, 63), (65, 64), (130, 77), (17, 128), (3, 255),
    (300, 256), (5, 257), (6, 510), (4, 777), (259, 1024), (3, 1027), (2, 2048), (5, 2050), (9, 4096), (2, 5001), (3, 8192),
    (2, 8196), (2, 16384), (3, 16387), (1, 20000), (2, 40001),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("shape", LAYER_NORMS, ids=lambda s: "x".join(map(str, s)))
def test_layer_norm_and_its_gradients(fg, hip, shape, bias):
    rows, dim = shape
    x, g = 2 + 3 * normal(6, rows, dim), normal(7, rows, dim)
    w, b = 1 + 0.1 * normal(8, dim), 0.1 * normal(9, dim) if bias else None
    tx, tw, tb = new(fg, x, True), new(fg, w, True), new(fg, b, True) if bias else None
    got = weighted(fg, tx.layer_norm(tw, tb), g, [t for t in (tx, tw, tb) if t])
    for name, a, (want, bound) in zip(("y", "dx", "dw", "db"), got, layer_norm64(x, w, b, g, 1e-5)):
        check(name, a, want, bound)
    assert np.array_equal(tx.layer_norm(tw, tb).numpy(), got[0])  # the same without the gradients


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim", [(3000, 8), (2500, 100), (1100, 520)])
def test_layer_norm_of_many_rows(fg, hip, rows, dim):
    x, g, w, b = 2 + 3 * normal(10, rows, dim), normal(11, rows, dim), 1 + 0.1 * normal(12, dim), normal(13, dim)
    tx, tw, tb = new(fg, x, True), new(fg, w, True), new(fg, b, True)
    got = weighted(fg, tx.layer_norm(tw, tb, eps=1e-3), g, [tx, tw, tb])
    for name, a, (want, bound) in zip(("y", "dx", "dw", "db"), got, layer_norm64(x, w, b, g, 1e-3)):
        check(name, a, want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [1, 6, 100, 3000])
def test_layer_norm_of_equal_numbers_is_the_bias(fg, hip, dim):
    # A mean of equal numbers is off by no more than its sum's roundings, which eps outweighs; of zeros by nothing.
    x = np.zeros((4, dim), np.float32)
    x[2:] = 3.0
    w, b, g = normal(14, dim), normal(15, dim), normal(16, 4, dim)
    tx, tw, tb = new(fg, x, True), new(fg, w, True), new(fg, b, True)
    y, dx, dw, db = weighted(fg, tx.layer_norm(tw, tb), g, [tx, tw, tb])
    assert np.array_equal(y[:2], np.broadcast_to(b, (2, dim)))
    off = 3.0 * (dim / 16 + 17) * U / 1e-5 ** 0.5
    assert np.abs(y[2:] - b).max() <= off * np.abs(w).max() + 2 * U * np.abs(b).max()
    assert np.isfinite(dx).all() and np.isfinite(dw).all()


@pytest.mark.gpu
def test_layer_norm_rows_keep_to_themselves(fg, hip):
    # A NaN or an infinity spoils its row and dw, and no other row; db sums the gradients alone.
    for dim in (40, 700, 9000):
        x, g, w = normal(17, 5, dim), normal(18, 5, dim), normal(19, dim)
        tw, tb = new(fg, w, True), new(fg, w, True)
        tx = new(fg, x, True)
        clean = weighted(fg, tx.layer_norm(tw, tb), g, [tx, tw, tb])
        for what in (np.nan, np.inf):
            bad = x.copy()
            bad[2, dim // 2] = what
            tx = new(fg, bad, True)
            y, dx, dw, db = weighted(fg, tx.layer_norm(tw, tb), g, [tx, tw, tb])
            rest = [0, 1, 3, 4]
            assert np.array_equal(y[rest], clean[0][rest]) and np.array_equal(dx[rest], clean[1][rest])
            assert np.isnan(y[2]).any() and np.isnan(dw).any() and np.array_equal(db, clean[3])


# ── the loss of token labels (GPU) ──────────────────────────────────────────


def loss64(x, labels, gout=1.0):
    """The loss and the logits' gradient, each with its bound. A term exp(x - top) is off by the rounding of its
    argument (three of |x - top|) and of the function (two steps), its sum by `deep` additions more; a logarithm by two
    steps, and a product."""
    x = x.astype(np.float64)
    rows, classes = x.shape
    valid = (labels >= 0) & (labels < classes)
    at, n = np.where(valid, labels, 0), max(1, int(valid.sum()))
    deep = classes / 16 + 16
    top = x.max(1, keepdims=True)
    a = np.where(np.isinf(x), 0.0, top - x)
    e = np.exp(x - top)
    ee = e * (3 * a + 6) * U
    s = e.sum(1, keepdims=True)
    es = ee.sum(1, keepdims=True) + deep * U * s
    picked = x[np.arange(rows), at][:, None]
    each = np.log(s) + top - picked
    eeach = es / s + 6 * U * np.abs(np.log(s)) + 3 * U * (np.abs(top - picked) + np.abs(each))
    loss = np.where(valid[:, None], each, 0).sum() / n
    eloss = np.where(valid[:, None], eeach, 0).sum() / n + 2 * U * abs(loss)
    p = e / s
    ep = ee / s + p * (es / s + 3 * U)
    one = np.zeros_like(x)
    one[np.arange(rows), at] = 1
    dx = np.where(valid[:, None], (p - one) * gout / n, 0.0)
    edx = np.where(valid[:, None], ep * abs(gout) / n, 0.0) + 4 * U * np.abs(dx)
    return (np.array([loss]), 1.1 * eloss), (dx, 1.1 * edx)


LOSSES = [  # rows, classes
    (1, 1), (1, 2), (3, 2), (256, 10), (5, 31), (64, 64), (7, 65), (33, 257), (130, 1000), (9, 1027), (300, 77), (4, 4096),
    (3, 5001), (2, 16384), (5, 16387), (3, 32768), (2, 32771), (2, 50001), (1, 70000), (2, 128000), (2000, 3),
    (2100, 9), (2500, 520),
    (3, 2017), (3, 2018), (40, 4099), (33, 8161), (3, 8162), (9, 32737), (2, 32738), (2, 65505), (2, 65506),
]


@pytest.mark.gpu
@pytest.mark.parametrize("ignored", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("shape", LOSSES, ids=lambda s: "x".join(map(str, s)))
def test_token_cross_entropy_and_its_gradient(fg, hip, shape, ignored):
    rows, classes = shape
    r = seeded(20)
    x = 3 * normal(21, rows, classes)
    labels = r.integers(0, classes, rows)
    labels = np.where(r.random(rows) < ignored, r.choice([-1, -100, classes, 2 ** 31 - 1, -(2 ** 31)], rows), labels).astype(np.int32)
    tx, tl = new(fg, x, True), new(fg, labels)
    want, dwant = loss64(x, labels)
    loss = tx.token_cross_entropy(tl)
    dx = loss.gradient([tx])[0]
    fg.Tensor.realize_many([loss, dx])
    check("loss", loss.numpy(), *want)
    check("dx", dx.numpy(), *dwant)
    # Alone, and under a gradient that is not 1.
    assert np.array_equal(tx.token_cross_entropy(tl).numpy(), loss.numpy())
    scaled = tx.token_cross_entropy(tl).mul(new(fg, np.array([-2.5], np.float32))).gradient([tx])[0]
    check("scaled", scaled.numpy(), *loss64(x, labels, -2.5)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(131072, 10), (70001, 33), (20001, 270), (17000, 1025)], ids=lambda s: "x".join(map(str, s)))
def test_token_cross_entropy_of_many_rows(fg, hip, shape):
    test_token_cross_entropy_and_its_gradient(fg, hip, shape, 0.4)


@pytest.mark.gpu
@pytest.mark.parametrize("classes", [9, 300, 20000, 60000])
def test_banned_classes_take_no_part(fg, hip, classes):
    # Logits of -inf and of the type's lowest value are classes of probability 0, wherever they are.
    x = 3 * normal(22, 6, classes)
    r = seeded(23)
    labels = r.integers(0, classes, 6).astype(np.int32)
    banned = r.random((6, classes)) < 0.4
    banned[0] = True  # the label alone is left
    banned[1, : classes - 2] = True
    banned[np.arange(6), labels] = False
    clean = np.where(banned, -1e4, x).astype(np.float32)
    want, dwant = loss64(clean, labels)
    for low in (-np.inf, np.finfo(np.float32).min):
        tx, tl = new(fg, np.where(banned, low, x).astype(np.float32), True), new(fg, labels)
        loss = tx.token_cross_entropy(tl)
        dx = loss.gradient([tx])[0]
        fg.Tensor.realize_many([loss, dx])
        check("loss", loss.numpy(), *want)
        check("dx", dx.numpy(), *dwant)
        assert not dx.numpy()[banned].any()


@pytest.mark.gpu
@pytest.mark.parametrize("classes", [9, 300, 20000, 60000])
def test_rows_of_no_class_and_rows_that_are_not_finite(fg, hip, classes):
    x, labels = 3 * normal(24, 5, classes), np.array([1, 2, -1, 4, 5], np.int32)
    clean = loss64(x, labels)[1]
    for what in (np.nan, np.inf, None):
        for row in (2, 3):
            bad = x.copy()
            if what is None:
                bad[row] = -np.inf
            else:
                bad[row, classes - 1] = what
            tx, tl = new(fg, bad, True), new(fg, labels)
            loss = tx.token_cross_entropy(tl)
            dx = loss.gradient([tx])[0]
            fg.Tensor.realize_many([loss, dx])
            loss, dx = loss.numpy(), dx.numpy()
            rest = [i for i in range(5) if i != row]
            check("dx", dx[rest], clean[0][rest], clean[1][rest])
            if row == 2:  # ignored, whatever it holds
                assert np.isfinite(loss).all() and not dx[2].any()
            else:
                assert np.isnan(loss).all() and np.isnan(dx[3]).any()


@pytest.mark.gpu
def test_large_logits_and_labels_of_all_rows(fg, hip):
    # Where exp itself would overflow or vanish; and the loss of one-hot rows.
    x = (normal(25, 40, 70) * np.float32(2.0) ** np.linspace(-30, 60, 40, dtype=np.float32)[:, None])
    labels = seeded(26).integers(0, 70, 40).astype(np.int32)
    tx, tl = new(fg, x, True), new(fg, labels)
    loss = tx.token_cross_entropy(tl)
    dx = loss.gradient([tx])[0]
    fg.Tensor.realize_many([loss, dx])
    want, dwant = loss64(x, labels)
    check("loss", loss.numpy(), *want)
    check("dx", dx.numpy(), *dwant)
    x = 3 * normal(27, 40, 70)
    tx, t1 = new(fg, x, True), new(fg, np.eye(70, dtype=np.float32)[labels])
    (want, bound), _ = loss64(x, labels)
    check("one-hot", tx.cross_entropy(t1).numpy().reshape(1), want, 4 * bound)


# ── norms and clipping (GPU) ────────────────────────────────────────────────


SHAPES = {
    "one": [(1,)], "classifier": [(128, 784), (128,), (10, 128), (10,)],
    "ragged": [(4095,), (4096,), (4097,), (3, 5, 7), (1, 1), (8192,), (12289,), (2, 2)],
    "16": [(1 + 37 * i,) for i in range(16)], "17": [(1 + 37 * i,) for i in range(17)], "64": [(1 + 37 * i,) for i in range(64)], "65": [(1 + 37 * i,) for i in range(65)],
    "200": [(3 + i % 5, 700) for i in range(200)],
}


@pytest.mark.gpu
@pytest.mark.parametrize("times", [0.25, 4.0])
@pytest.mark.parametrize("name", SHAPES)
def test_clip_norm(fg, hip, name, times):
    xs = [normal(30 + i, *s) for i, s in enumerate(SHAPES[name])]
    norm = np.sqrt(sum((x.astype(np.float64) ** 2).sum() for x in xs))
    got, clipped = fg.clip_norm([new(fg, x) for x in xs], times * norm)
    fg.Tensor.realize_many([got] + clipped)
    # Sums are in 64 bits: the norm is rounded once, and so is the scale.
    check("norm", got.numpy(), np.array([norm]), 1.01 * U * norm)
    for x, y in zip(xs, clipped):
        want = x.astype(np.float64) * min(1.0, times)
        check("clipped", y.numpy(), want, 2.01 * U * np.abs(want))
    check("norm alone", fg.global_norm([new(fg, x) for x in xs]).numpy(), np.array([norm]), 1.01 * U * norm)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-42, 1e-30, 1e18, 3e33])
def test_clip_norm_of_small_and_large_values(fg, hip, size):
    # Squares of these leave float32's range.
    xs = [(normal(31, 5000) * size).astype(np.float32), (normal(32, 3) * size).astype(np.float32)]
    norm = np.sqrt(sum((x.astype(np.float64) ** 2).sum() for x in xs))
    got, clipped = fg.clip_norm([new(fg, x) for x in xs], 0.5 * norm)
    fg.Tensor.realize_many([got] + clipped)
    step = 2.0 ** -149  # of numbers below TINY
    check("norm", got.numpy(), np.array([norm]), 1.01 * U * norm + step)
    for x, y in zip(xs, clipped):
        want = 0.5 * x.astype(np.float64)
        check("clipped", y.numpy(), want, 2.01 * U * np.abs(want) + step)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_replayed_clips_of_many_tensors(fg, hip, graphs):
    with graphs_on(fg, 2 if graphs else 0):
        fg.clear_caches()
        for turn in range(5):
            xs = [(turn + 1) * normal(200 + 7 * turn + i, 5 + 61 * i) for i in range(70)]
            norm = np.sqrt(sum((x.astype(np.float64) ** 2).sum() for x in xs))
            got, clipped = fg.clip_norm([new(fg, x) for x in xs], 2.0)
            fg.Tensor.realize_many(clipped + [got])
            new(fg, normal(60, 1000)).exp().numpy()  # other work in between
            check("norm", got.numpy(), np.array([norm]), 1.01 * U * norm)
            for x, y in zip(xs, clipped):
                check("clipped", y.numpy(), x * (2.0 / norm), 2.01 * U * np.abs(x * (2.0 / norm)))


@pytest.mark.gpu
def test_clipped_gradients_are_clipped_again_and_added_to(fg, hip):
    p = new(fg, normal(280, 40), True)
    w = new(fg, normal(281, 40))
    opt = fg.Sgd([p], 0.5)
    g = w.numpy().astype(np.float64)
    size = np.linalg.norm(g)
    p.mul(w).sum([0]).backward()
    first = opt.clip_grad_norm(1.0)
    second = opt.clip_grad_norm(0.5)
    check("first", first.numpy(), np.array([size]), 2 * U * size)
    check("second", second.numpy(), np.array([1.0]), np.array([6 * U]))
    p.mul(w).sum([0]).backward()  # gradients add up
    want = g * (1 + 0.5 / size)
    check("sum", p.grad().numpy(), want, 8 * U * np.abs(want))
    before = p.numpy().astype(np.float64)
    opt.step()
    check("step", p.numpy(), before - 0.5 * want, 2 * U * (np.abs(before) + 10 * np.abs(want)))


@pytest.mark.gpu
def test_clip_norm_of_zeros_and_of_what_is_not_finite(fg, hip):
    x, y = np.zeros(700, np.float32), normal(33, 5000)
    norm, (a,) = fg.clip_norm([new(fg, x)], 1.0)
    assert norm.numpy()[0] == 0 and not a.numpy().any()
    bad = y.copy()
    bad[4999] = np.nan
    norm, (a, b) = fg.clip_norm([new(fg, x), new(fg, bad)], 1.0)
    assert np.isnan(norm.numpy()).all() and np.isnan(a.numpy()).all() and np.isnan(b.numpy()).all()
    bad[4999] = np.inf
    norm, (a, b) = fg.clip_norm([new(fg, y), new(fg, bad)], 1.0)
    assert np.isinf(norm.numpy()).all() and not a.numpy().any() and np.isnan(b.numpy()[4999]) and not b.numpy()[:4999].any()


@pytest.mark.gpu
def test_the_same_tensor_twice_counts_twice(fg, hip):
    x = normal(34, 300)
    t = new(fg, x)
    norm, clipped = fg.clip_norm([t, t.reshape([30, 10]), t], 1.0)
    fg.Tensor.realize_many([norm] + clipped)
    want = np.sqrt(3 * (x.astype(np.float64) ** 2).sum())
    check("norm", norm.numpy(), np.array([want]), 1.01 * U * want)
    for c in clipped:
        check("clipped", c.numpy().reshape(-1), x / want, 2.01 * U * np.abs(x / want))


# ── together (GPU) ──────────────────────────────────────────────────────────


def every_call(fg, seed):
    """One of each call with its gradients, as tensors to realise, and their inputs as arrays."""
    w, ids, g = normal(seed, 50, 24), seeded(seed).integers(0, 50, 90).astype(np.int32), normal(seed + 1, 90, 24)
    n, b = normal(seed + 2, 24), normal(seed + 3, 24)
    tw, tn, tb = new(fg, w, True), new(fg, n, True), new(fg, b, True)
    h = tw.embedding(new(fg, ids), 2.0).layer_norm(tn, tb)
    logits = h.add(new(fg, g))
    loss = logits.token_cross_entropy(new(fg, (ids % 24).astype(np.int32)))
    grads = loss.gradient([tw, tn, tb])
    norm, clipped = fg.clip_norm(grads, 0.01)
    return [h, loss, norm] + grads + clipped


@pytest.mark.gpu
def test_the_same_inputs_give_the_same_bits(fg, hip):
    def run():
        outs = every_call(fg, 40)
        fg.Tensor.realize_many(outs)
        return [t.numpy() for t in outs]

    first = run()
    for _ in range(3):
        assert all(np.array_equal(a, b) for a, b in zip(run(), first))


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_replayed_calls_read_the_new_inputs(fg, hip, graphs):
    eager = []
    for seed in (50, 51, 52, 53):
        fg.clear_caches()
        outs = every_call(fg, seed)
        fg.Tensor.realize_many(outs)
        eager.append([t.numpy() for t in outs])
    with graphs_on(fg, 2 if graphs else 0):
        fg.clear_caches()
        for seed, want in list(zip((50, 51, 52, 53), eager)) * 2:
            outs = every_call(fg, seed)
            fg.Tensor.realize_many(outs)
            fg.synchronize("hip")
            new(fg, normal(60, 1000)).exp().numpy()  # other work in between
            assert all(np.array_equal(t.numpy(), x) for t, x in zip(outs, want))


@pytest.mark.gpu
def test_calls_read_views_literals_and_what_an_update_replaces(fg, hip):
    w, ids = normal(61, 8, 12), np.array([3, 0, 7, 7, 1, 2], np.int32)
    tw, ti = new(fg, w), new(fg, ids)
    t = tw.permute([1, 0])  # a view: its rows are w's columns
    assert np.array_equal(t.embedding(ti.narrow(0, 1, 3)).numpy(), w.T[ids[1:4]])
    assert np.array_equal(fg.Tensor.ones([8, 4], "hip").embedding(ti).numpy(), np.ones((6, 4), np.float32))
    part = tw.narrow(0, 2, 4)
    (want, bound), *_ = layer_norm64(w[2:6], np.ones(12), None, np.zeros((4, 12)), 1e-5)
    check("narrow", part.layer_norm(fg.Tensor.ones([12], "hip")).numpy(), want, bound)
    zeros = fg.Tensor.zeros([12], "hip")
    check("zero bias", part.layer_norm(fg.Tensor.ones([12], "hip"), zeros).numpy(), want, bound)
    p = new(fg, w)
    before = p.embedding(ti)
    p.assign(p.add(p))
    fg.Tensor.realize_many([before, p])
    assert np.array_equal(before.numpy(), w[ids]) and np.array_equal(p.embedding(ti).numpy(), 2 * w[ids])
    norm, (c,) = fg.clip_norm([tw.narrow(1, 0, 5)], 1e9)
    assert np.array_equal(c.numpy(), w[:, :5])


@pytest.mark.gpu
def test_gradients_of_gradients_and_of_norms_are_refused(fg, hip):
    tw, tn = new(fg, normal(62, 5, 6), True), new(fg, normal(63, 6), True)
    ids = new(fg, np.array([1, 2, 2], np.int32))
    for loss in (tw.embedding(ids).mul(tw.embedding(ids)).sum([0, 1]), tw.layer_norm(tn).mul(tw).sum([0, 1]),
                 tw.token_cross_entropy(new(fg, np.zeros(5, np.int32)))):
        g = loss.gradient([tw])[0]
        with pytest.raises(fg.FerrogradError, match="gradient not implemented"):
            (g if g.numel() == 1 else g.sum([0, 1])).gradient([tw])
    with pytest.raises(fg.FerrogradError, match="gradient not implemented"):
        fg.global_norm([tw]).gradient([tw])


@pytest.mark.gpu
def test_gradients_against_differences(fg, hip):
    # The loss of a small model, and its slope along a direction by central differences in float64 on the host.
    ids, labels = np.array([0, 4, 4, 2, -1, 1], np.int32), np.array([1, 0, 3, -5, 2, 2], np.int32)
    params = [normal(64, 5, 16), 1 + 0.1 * normal(65, 16), 0.1 * normal(66, 16), normal(67, 4, 16)]

    def loss(ps):
        w, n, b, out = ps
        h = np.where(((ids >= 0) & (ids < 5))[:, None], w[np.clip(ids, 0, 4)] * 1.5, 0.0)
        c = h - h.mean(1, keepdims=True)
        z = (c / np.sqrt((c * c).mean(1, keepdims=True) + 1e-5) * n + b) @ out.T
        keep = labels >= 0
        lse = np.log(np.exp(z).sum(1))
        return (lse - z[np.arange(6), np.clip(labels, 0, 3)])[keep].mean()

    ts = [new(fg, p, True) for p in params]
    z = ts[0].embedding(new(fg, ids), 1.5).layer_norm(ts[1], ts[2]).matmul(ts[3].permute([1, 0]))
    grads = [g.numpy().astype(np.float64) for g in z.token_cross_entropy(new(fg, labels)).gradient(ts)]
    wide = [p.astype(np.float64) for p in params]
    for seed in range(4):
        ds = [seeded(70 + seed).standard_normal(p.shape) for p in params]
        step = 1e-5
        slope = (loss([p + step * d for p, d in zip(wide, ds)]) - loss([p - step * d for p, d in zip(wide, ds)])) / (2 * step)
        terms = [(g * d) for g, d in zip(grads, ds)]
        # The difference is off by step^2 times a third derivative of order 10; the gradients by a few hundred roundings.
        assert abs(sum(t.sum() for t in terms) - slope) <= 1e-8 + 500 * U * sum(np.abs(t).sum() for t in terms)


@pytest.mark.gpu
def test_a_loss_and_what_is_made_of_it_beside_its_gradient(fg, hip):
    # The gradient's call makes the loss, for its own readers too, whichever is realised first.
    x, labels = 3 * normal(90, 30, 40), seeded(91).integers(0, 40, 30).astype(np.int32)
    tx, tl, two = new(fg, x, True), new(fg, labels), new(fg, np.array([2.0], np.float32))
    (want, bound), (dwant, dbound) = loss64(x, labels)
    loss = tx.token_cross_entropy(tl)
    double, dx = loss.mul(two), loss.gradient([tx])[0]
    got = classes(fg, [double, dx])
    assert "token_loss" not in got and got.count("token_loss_grad") == 1
    fg.Tensor.realize_many([double, dx])
    assert loss.is_realized()
    check("double", double.numpy(), 2 * want, 2.1 * bound)
    check("dx", dx.numpy(), dwant, dbound)
    # Only the gradient: the loss is there as well.
    loss = tx.token_cross_entropy(tl)
    dx = loss.gradient([tx])[0].realize()
    assert loss.is_realized()
    check("loss", loss.numpy(), want, bound)
    # The loss first, then its gradient; a gradient through a function of the loss.
    loss = tx.token_cross_entropy(tl)
    dx = loss.gradient([tx])[0]
    check("loss", loss.numpy(), want, bound)
    check("dx", dx.numpy(), dwant, dbound)
    loss = tx.token_cross_entropy(tl)
    square = loss.mul(loss)
    dsq = square.gradient([tx])[0]
    fg.Tensor.realize_many([dsq, square, loss])
    check("square", square.numpy(), want * want, 2.2 * bound * want)
    check("dsq", dsq.numpy(), 2 * want * dwant, 2.2 * (want * dbound + bound * np.abs(dwant)) + 4 * U * np.abs(2 * want * dwant))


@pytest.mark.gpu
def test_weights_read_twice_and_gradients_that_are_broadcast(fg, hip):
    w, a, b = normal(92, 9, 6), np.array([1, 2, 2, 8], np.int32), np.array([2, 0, 5, 5], np.int32)
    tw = new(fg, w, True)
    y = tw.embedding(new(fg, a)).add(tw.embedding(new(fg, b), 2.0))
    dw = y.sum([0, 1]).gradient([tw])[0].numpy()
    want = np.bincount(a, minlength=9) + 2.0 * np.bincount(b, minlength=9)
    assert np.array_equal(dw, np.repeat(want[:, None], 6, 1))
    x, n = normal(93, 5, 6), normal(94, 6)
    tx, tn = new(fg, x, True), new(fg, n, True)
    y = tx.layer_norm(tn, tn)  # one tensor as weight and bias
    dx, dn = (t.numpy() for t in y.sum([0, 1]).gradient([tx, tn]))
    _, (wx, ex), (ww, ew), (wb, eb) = layer_norm64(x, n, n, np.ones((5, 6), np.float32), 1e-5)
    check("dx", dx, wx, ex)
    check("dn", dn, ww + wb, ew + eb + U * np.abs(ww + wb))


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [None, 0.05])
def test_a_train_step_takes_labels_and_clips(fg, hip, max_norm):
    from ferrograd_amd.mlp import Mlp, synthetic_batch, train_step

    xs, ts = synthetic_batch(64, 20, 7, 1, 2)
    labels = ts.argmax(1).astype(np.int32)
    got = []
    for targets in (ts, labels):
        fg.reset_init_seed(11)
        model = Mlp((20, 16, 7), hip)
        params = model.parameters()
        before = [p.numpy().astype(np.float64) for p in params]
        loss = train_step(model, fg.Sgd(params, 0.5), new(fg, xs), new(fg, targets), max_norm=max_norm)
        got.append([loss.numpy().reshape(-1)] + [(b - p.numpy()) / 0.5 for p, b in zip(params, before)])
    # The same step, by sums in other orders: a few hundred roundings of terms no larger than their sums' norms.
    for a, b, p in zip(*got, [np.zeros(1)] + before):
        assert np.linalg.norm(a - b) <= 500 * U * np.linalg.norm(b) + 4 * U * np.linalg.norm(p) / 0.5
    norm = np.sqrt(sum((g ** 2).sum() for g in got[1][1:]))
    assert norm > 0.06 if max_norm is None else abs(norm - max_norm) <= 1e-5


# Larger tensors than generated kernels make are made of a few rows by embedding,
# and their rows read by it again.


@pytest.mark.gpu
def test_ids_of_four_passes_and_rows_past_32_bits(fg, hip):
    # 2^30 ids, whose keys have 31 bits.
    tokens = 17000
    ids = seeded(95).integers(0, 1 << 30, tokens).astype(np.int32)
    ids[:9] = [0, (1 << 30) - 1, 7, 7, 1 << 30, -1, (1 << 30) - 1, 12345678, 7]
    g = normal(96, tokens, 1)
    w = fg.Tensor.zeros([1 << 30, 1], "hip").with_requires_grad(True)
    dw = w.embedding(new(fg, ids)).mul(new(fg, g)).sum([0, 1]).gradient([w])[0].realize()
    inside = (ids >= 0) & (ids < 1 << 30)
    names, at = np.unique(ids[inside], return_inverse=True)
    want, size = np.zeros(len(names)), np.zeros(len(names))
    np.add.at(want, at, g[inside, 0].astype(np.float64))
    np.add.at(size, at, np.abs(g[inside, 0]))
    check("dw", dw.embedding(new(fg, names.astype(np.int32))).numpy()[:, 0], want, 4 * U * size)
    total = np.sqrt((want ** 2).sum())
    check("norm", fg.global_norm([dw]).numpy(), np.array([total]), 5 * U * total)  # all other rows are 0
    del w, dw
    # A weight of 2^32 elements and more: its last rows are read and written.
    rows, dim = (1 << 22) + 5, 1028
    table, which = np.stack([np.ones(dim), np.arange(dim)]).astype(np.float32), np.zeros(rows, np.int32)
    which[-1] = 1
    w = new(fg, table).embedding(new(fg, which)).realize().detach().with_requires_grad(True)
    ids = np.array([rows - 1, 3, rows - 2, rows - 1], np.int32)
    g = normal(97, 4, dim)
    y = w.embedding(new(fg, ids))
    dw = y.mul(new(fg, g)).sum([0, 1]).gradient([w])[0]
    fg.Tensor.realize_many([y, dw])
    assert np.array_equal(y.numpy(), table[[1, 0, 0, 1]])
    want = np.stack([g[0].astype(np.float64) + g[3], g[2], g[1]])
    check("dw", dw.embedding(new(fg, np.array([rows - 1, rows - 2, 3], np.int32))).numpy(), want, U * np.abs(want))
    total = np.sqrt((want ** 2).sum())
    check("norm", fg.global_norm([dw]).numpy(), np.array([total]), 3 * U * total)


@pytest.mark.gpu
def test_rows_of_matrices_past_32_bits(fg, hip):
    rows, cols = (1 << 21) + 3, 2052  # over 2^32 elements
    last, which = normal(98, 2, cols), np.zeros(rows, np.int32)
    which[-2:] = [1, 2]
    table = np.concatenate([np.ones((1, cols), np.float32), last])
    x = new(fg, table).embedding(new(fg, which)).realize().detach().with_requires_grad(True)
    ends = new(fg, np.array([0, rows - 2, rows - 1], np.int32))
    w, b = normal(99, cols), normal(100, cols)
    y = x.layer_norm(new(fg, w), new(fg, b)).realize().embedding(ends).numpy()
    (want, bound), *_ = layer_norm64(table, w, b, np.zeros_like(table), 1e-5)
    check("y", y, want, bound)
    labels = np.full(rows, -1, np.int32)
    labels[-2:] = [7, 2051]
    loss = x.token_cross_entropy(new(fg, labels))
    dx = loss.gradient([x])[0]
    fg.Tensor.realize_many([loss, dx])
    (want, bound), (dwant, dbound) = loss64(last, labels[-2:])
    check("loss", loss.numpy(), want, bound)
    got = dx.embedding(ends).numpy()
    check("dx", got[1:], dwant, dbound)
    total = np.sqrt((dwant ** 2).sum())
    check("all", fg.global_norm([dx]).numpy(), np.array([total]), np.sqrt((dbound ** 2).sum()) + U * total)
    del dx, loss
    norm, (c,) = fg.clip_norm([x], 1.0)
    total = np.sqrt((rows - 2) * float(cols) + (last.astype(np.float64) ** 2).sum())
    check("clipped", c.embedding(ends).numpy(), table / total, 2.01 * U * np.abs(table / total))
    check("norm", norm.numpy(), np.array([total]), 1.01 * U * total)


def model64(torch, ps, ids, labels, pos, heads, batch):
    from test_operators import Torch64

    table, nw, nb, wq, wk, wv, wo, qn, kn, fw, fb = ps
    inside = (ids >= 0) & (ids < table.shape[0])
    x = torch.where(inside[:, None], table[torch.where(inside, ids, 0)] * 4.0, 0.0)

    def norm(z, w, b):
        c = z - z.mean(1, keepdim=True)
        return c / ((c * c).mean(1, keepdim=True) + 1e-5).sqrt() * w + b

    z = norm(x, nw, nb)
    q, k = (Torch64.norm_rotate(z @ w.T, n, pos, heads, 1e-6, 10000.0) for w, n in ((wq, qn), (wk, kn)))
    x = x + Torch64.attention(q, k, z @ wv.T, heads, heads, batch, torch.full((batch,), len(ids) // batch)) @ wo.T
    logits = norm(x, fw, fb) @ table.T  # the embedding's own rows
    keep = (labels >= 0) & (labels < table.shape[0])
    return torch.nn.functional.cross_entropy(logits[keep], labels[keep])


@pytest.mark.gpu
def test_a_token_model_has_the_loss_the_norm_and_the_updates_of_its_parameters(fg, hip):
    # Embedding, norms, attention, the embedding's rows again as classes, the loss of the next tokens, clipping.
    import torch

    from ferrograd_amd.attention import SelfAttention

    vocab, dim, heads, batch, n, lr = 37, 32, 4, 3, 21, 0.5
    fg.reset_init_seed(9)
    embed, first, last = fg.Embedding(vocab, dim, hip, scale=4.0), fg.LayerNorm(dim, hip), fg.LayerNorm(dim, hip)
    layer = SelfAttention(dim, heads, device=hip)
    params = embed.parameters() + first.parameters() + layer.parameters() + last.parameters()
    opt = fg.Sgd(params, lr)
    pos = np.tile(np.arange(n, dtype=np.int32), batch)
    r = seeded(80)
    tol = 3 * 9 * 16 * (2 * dim + n + batch * n + vocab) * U  # as for a layer of attention, and its roundings
    for step in range(3):
        tokens = r.integers(0, vocab, (batch, n + 1)).astype(np.int32)
        tokens[1, 15:] = -1  # padding
        ids, labels = tokens[:, :-1].reshape(-1).copy(), tokens[:, 1:].reshape(-1).copy()
        before = [p.numpy().astype(np.float64) for p in params]
        x = embed(new(fg, ids))
        x = x.add(layer(first(x), new(fg, pos), batch))
        loss = last(x).matmul(embed.weight.permute([1, 0])).token_cross_entropy(new(fg, labels))
        opt.zero_grad()
        loss.backward()
        norm = opt.clip_grad_norm(0.1)
        opt.step()
        ps = [torch.tensor(p, requires_grad=True) for p in before]
        want = model64(torch, ps, torch.tensor(ids).long(), torch.tensor(labels).long(), torch.tensor(pos), heads, batch)
        grads = [g.numpy() for g in torch.autograd.grad(want, ps)]
        total = np.sqrt(sum((g ** 2).sum() for g in grads))
        want = float(want.detach())
        assert abs(float(loss.to_vec()[0]) - want) <= tol * abs(want), step
        assert abs(float(norm.to_vec()[0]) - total) <= tol * total, step
        assert total > 0.1  # it is clipped
        for i, (p, b, g) in enumerate(zip(params, before, grads)):
            update, g = (b - p.numpy()) / lr, g * (0.1 / total)
            rounding = U * np.linalg.norm(b) / lr
            assert np.linalg.norm(update - g) <= tol * (np.linalg.norm(g) + 0.1) + 2 * rounding, (step, i)
