"""Attention, per-head norms with the position rotation, and dropout: calls side
by side on the same tensors, values that are not finite or of very unlike sizes,
and the largest sizes."""
import numpy as np
import pytest

import attention_ref
from attention_ref import U
from conftest import graphs_on, seeded
from test_operators import attention_inputs, check, new, norm_rotate_ref


# ── calls on the same tensors that differ in a parameter only ───────────────


def lazy(fg, *shape, dtype=None):
    t = fg.Tensor.zeros(list(shape), "hip") if dtype is None else fg.Tensor.zeros(list(shape), "hip", dtype)
    return t.with_requires_grad(True) if dtype is None else t


def written_twice(fg, roots):
    """Buffers of the plan of `roots` that more than one call writes."""
    items = fg.debug_plan(roots, fuse=True, render_hip=True)["items"]
    storage = {it["output"] for it in items if it["class"] == "storage"}
    writers = {}
    for it in items:
        last = it["inputs"][-{"attention": 1, "attention_grad": 2, "norm_rotate_grad": 1}.get(it["class"], 0):] \
            if it["class"] in ("attention", "attention_grad", "norm_rotate_grad") else []
        for a in last:
            assert a["buffer"] in storage
            writers[a["buffer"]] = writers.get(a["buffer"], 0) + 1
    assert writers
    return [b for b, n in writers.items() if n > 1]


@pytest.mark.parametrize("kw", [dict(causal=True), dict(scale=0.5), dict(batch=2)])
def test_attention_calls_that_differ_in_a_parameter_have_their_own_outputs(fg, kw):
    x = lazy(fg, 6, 8)
    y = x.attention(x, x, heads=2).add(x.attention(x, x, heads=2, **kw))
    assert not written_twice(fg, [y, y.sum([0, 1]).gradient([x])[0]])


@pytest.mark.parametrize("kw", [dict(eps=1e-3), dict(base=500000.0)])
def test_norms_that_differ_in_a_parameter_have_their_own_outputs(fg, kw):
    x, w, pos = lazy(fg, 6, 8), lazy(fg, 4), lazy(fg, 6, dtype=fg.I32)
    y = x.norm_rotate(w, pos, heads=2).add(x.norm_rotate(w, pos, heads=2, **kw))
    assert not written_twice(fg, [y, *y.sum([0, 1]).gradient([x, w])])


def both(a, b):
    """(value, bound) of the float32 sum of two results."""
    return a[0] + b[0], a[1] + b[1] + 2 * U * (np.abs(a[0]) + np.abs(b[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(causal=True), dict(scale=0.5), dict(batch=2)])
@pytest.mark.parametrize("graphs", [False, True])
def test_gradients_of_two_attention_calls_on_the_same_tensors(fg, hip, kw, graphs):
    import contextlib

    with graphs_on(fg) if graphs else contextlib.nullcontext():
        for step in range(3):
            q, k, v, g = attention_inputs(50 + step, 1, 90, 90, 4, 2, 32)
            tq, tk, tv = (new(fg, t, True) for t in (q, k, v))
            y = tq.attention(tk, tv, heads=4, kv_heads=2).add(tq.attention(tk, tv, heads=4, kv_heads=2, **kw))
            grads = y.mul(new(fg, g)).sum([0, 1]).gradient([tq, tk, tv])
            fg.Tensor.realize_many([y, *grads])
            a = attention_ref.attention(q, k, v, 1, 4, 2, g=g)
            b = attention_ref.attention(q, k, v, heads=4, kv_heads=2, g=g, **{"batch": 1, **kw})
            for name, t in zip(("y", "dq", "dk", "dv"), (y, *grads)):
                check((step, name), t.numpy(), *both(a[name], b[name]))


@pytest.mark.gpu
def test_gradients_of_an_attention_call_after_another_on_the_same_tensors_ran(fg, hip):
    q, k, v, g = attention_inputs(54, 1, 90, 90, 4, 4, 32)
    tq, tk, tv = (new(fg, t, True) for t in (q, k, v))
    a, b = tq.attention(tk, tv, heads=4), tq.attention(tk, tv, heads=4, causal=True)
    tg = new(fg, g)
    da, db = (t.mul(tg).sum([0, 1]).gradient([tq, tk, tv]) for t in (a, b))
    a.realize()
    b.realize()
    for grads, causal in ((da, False), (db, True)):
        want = attention_ref.attention(q, k, v, 1, 4, 4, causal=causal, g=g)
        for name, t in zip(("dq", "dk", "dv"), grads):
            check(name, t.numpy(), *want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(eps=1e-3), dict(base=500000.0)])
def test_gradients_of_two_norms_on_the_same_tensors(fg, hip, kw):
    r = seeded(55)
    x = (3 * r.standard_normal((37, 3 * 16))).astype(np.float32)
    w = (1 + 0.3 * r.standard_normal(16)).astype(np.float32)
    g = r.standard_normal(x.shape).astype(np.float32)
    pos = r.integers(0, 4096, 37).astype(np.int32)
    a = norm_rotate_ref(x, w, pos, 3, 1e-6, 10000.0, g)
    b = norm_rotate_ref(x, w, pos, 3, **{"eps": 1e-6, "base": 10000.0, **kw}, g=g)
    tx, tw, tp = new(fg, x, True), new(fg, w, True), new(fg, pos)
    for step in range(2):
        y = tx.norm_rotate(tw, tp, 3).add(tx.norm_rotate(tw, tp, 3, **kw))
        dx, dw = y.mul(new(fg, g)).sum([0, 1]).gradient([tx, tw])
        fg.Tensor.realize_many([y, dx, dw])
        for name, t in (("y", y), ("dx", dx), ("dweight", dw)):
            check((step, name), t.numpy(), *both(a[name], b[name]))


# ── NaN and infinities that are seen ────────────────────────────────────────

# batch, sq, sk, heads, kv_heads, dim, lengths, and the launches of the forward pass
PATHS = {
    "small": (2, 3, 200, 4, 2, 24, None, ["token"]),
    "small in parts": (2, 1, 3000, 4, 2, 24, None, ["token", "join"]),
    "three columns in parts": (1, 1, 1300, 1, 1, 3, None, ["token", "join"]),
    "parts of one length": (10, 1, 2500, 12, 6, 24, [2500, 0, 2400, 1300, 2, 128, 129, 2499, 1, 2500], ["token", "join"]),
    "large": (4, 130, 257, 32, 32, 40, None, ["pack", "tiles"]),
    "large in parts": (1, 256, 4000, 16, 8, 64, None, ["pack", "tiles", "join"]),
}


def forward_launches(fg, batch, sq, sk, heads, kv_heads, dim, lengths, causal=False):
    q, k = fg.Tensor.zeros([batch * sq, heads * dim], "hip"), fg.Tensor.zeros([batch * sk, kv_heads * dim], "hip")
    y = q.attention(k, k, heads=heads, kv_heads=kv_heads, batch=batch, causal=causal,
                    lengths=None if lengths is None else fg.Tensor.zeros([batch], "hip", fg.I32))
    call = [it for it in fg.debug_plan([y], fuse=True, render_hip=True)["items"] if it["class"] == "attention"]
    return [l["name"].split("_")[2] for it in call for l in it["launches"]]


@pytest.mark.parametrize("path", PATHS)
def test_the_shapes_below_take_their_paths(fg, path):
    *shape, launches = PATHS[path]
    assert forward_launches(fg, *shape) == launches


def run_both(fg, q, k, v, g, **kw):
    """y and the gradients of attention, as arrays."""
    tq, tk, tv = (new(fg, t, True) for t in (q, k, v))
    if kw.get("lengths") is not None:
        kw["lengths"] = new(fg, np.asarray(kw["lengths"], np.int32))
    y = tq.attention(tk, tv, **kw)
    grads = y.mul(new(fg, g)).sum([0, 1]).gradient([tq, tk, tv])
    fg.Tensor.realize_many([y, *grads])
    return {n: t.numpy() for n, t in zip(("y", "dq", "dk", "dv"), (y, *grads))}


@pytest.mark.gpu
@pytest.mark.parametrize("what", [np.nan, np.inf], ids=["nan", "inf"])
@pytest.mark.parametrize("path", PATHS)
def test_rows_that_see_a_key_that_is_not_finite_are_not_finite(fg, hip, path, what):
    batch, sq, sk, heads, kv_heads, dim, lengths, _ = PATHS[path]
    kw = dict(batch=batch, heads=heads, kv_heads=kv_heads, lengths=lengths)
    q, k, v, g = attention_inputs(60, batch, sq, sk, heads, kv_heads, dim)
    q[:sq, 0] = np.abs(q[:sq, 0]) + 0.1  # an infinite key scores +infinity
    clean = run_both(fg, q, k, v, g, **kw)
    at = sk * 3 // 5
    k[at, 0] = what  # a visible key of the first sequence and key head
    got = run_both(fg, q, k, v, g, **kw)
    group = heads // kv_heads
    for name, rows, cols in (("y", sq, dim if what == np.inf else group * dim), ("dq", sq, dim), ("dk", sk, dim), ("dv", sk, dim)):
        bad = np.zeros(got[name].shape, bool)
        bad[:rows, :cols] = True
        assert not np.isfinite(got[name][bad]).any(), name
        rest = np.ones(got[name].shape, bool)  # what other key heads and sequences see
        rest[:rows, :(group if name in ("y", "dq") else 1) * dim] = False
        assert np.array_equal(got[name][rest], clean[name][rest]), name


@pytest.mark.gpu
@pytest.mark.parametrize("path", PATHS)
def test_a_query_that_is_nan_has_a_row_of_nan(fg, hip, path):
    batch, sq, sk, heads, kv_heads, dim, lengths, _ = PATHS[path]
    kw = dict(batch=batch, heads=heads, kv_heads=kv_heads, lengths=lengths)
    q, k, v, g = attention_inputs(61, batch, sq, sk, heads, kv_heads, dim)
    clean = run_both(fg, q, k, v, g, **kw)
    at = sq // 2
    q[at, dim - 1] = np.nan  # of the first sequence and head
    got = run_both(fg, q, k, v, g, **kw)
    bad = np.zeros(q.shape, bool)
    bad[at, :dim] = True
    assert np.isnan(got["y"][bad]).all() and np.isnan(got["dq"][bad]).all()
    assert np.array_equal(got["y"][~bad], clean["y"][~bad])
    seen = np.zeros(k.shape, bool)
    seen[:sk, :dim] = True
    for name in ("dk", "dv"):
        assert np.isnan(got[name][seen]).all(), name
        assert np.array_equal(got[name][~seen], clean[name][~seen]), name


@pytest.mark.gpu
@pytest.mark.parametrize("path", PATHS)
def test_a_value_that_is_nan_makes_its_column_nan(fg, hip, path):
    batch, sq, sk, heads, kv_heads, dim, lengths, _ = PATHS[path]
    kw = dict(batch=batch, heads=heads, kv_heads=kv_heads, lengths=lengths)
    q, k, v, g = attention_inputs(62, batch, sq, sk, heads, kv_heads, dim)
    v[sk // 2, 1] = np.nan
    got = run_both(fg, q, k, v, g, **kw)
    group = heads // kv_heads
    assert np.isnan(got["y"][:sq].reshape(sq, heads, dim)[:, :group, 1]).all()
    assert np.isnan(got["dq"][:sq, :group * dim]).all() and np.isnan(got["dk"][:sk, :dim]).all()
    rest = np.ones(q.shape, bool)
    rest[:sq, :group * dim] = False
    assert np.isfinite(got["y"][rest]).all() and np.isfinite(got["dq"][rest]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("path", [p for p in PATHS if PATHS[p][6] is None])
def test_a_key_that_scores_minus_infinity_weighs_nothing(fg, hip, path):
    batch, sq, sk, heads, kv_heads, dim, _, _ = PATHS[path]
    q, k, v, _ = attention_inputs(64, batch, sq, sk, heads, kv_heads, dim)
    q[:, ::dim] = np.abs(q[:, ::dim]) + 0.1
    rest = np.arange(batch * sk) % sk != sk // 4
    want = attention_ref.attention(q, k[rest], v[rest], batch, heads, kv_heads)["y"]
    k.reshape(batch, sk, kv_heads, dim)[:, sk // 4, :, 0] = -np.inf
    check("y", new(fg, q).attention(new(fg, k), new(fg, v), heads=heads, kv_heads=kv_heads, batch=batch).numpy(), *want)


# ── values of unlike sizes ──────────────────────────────────────────────────


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e20, 1e26, 1e30])
@pytest.mark.parametrize("zeros", ["last", "first", "between"])
def test_values_of_zero_beside_large_ones_take_their_probability(fg, hip, size, zeros):
    batch, sq, sk, heads, kv_heads, dim, lengths, _ = PATHS["large"]
    q, k, v, g = attention_inputs(63, batch, sq, sk, heads, kv_heads, dim, spread=0.5)
    v = (v * np.float32(size)).reshape(batch, sk, -1)
    v[:, {"last": slice(128, None), "first": slice(0, 128), "between": slice(64, 192)}[zeros]] = 0
    v = v.reshape(batch * sk, -1)
    g /= np.float32(size)
    kw = dict(batch=batch, heads=heads, kv_heads=kv_heads)
    got, want = run_both(fg, q, k, v, g, **kw), attention_ref.attention(q, k, v, g=g, **kw)
    for name in want:
        check(name, got[name], *want[name])


# What a query does not see, or weighs with nothing, and columns beside large
# ones: each against the call without the large numbers, whose values and bounds
# are those of numbers of one size.

UNLIKE = {  # batch, sq, sk, heads, kv_heads, dim
    "small": (1, 100, 100, 2, 1, 24),
    "large": (4, 200, 257, 32, 32, 40),
    "large in parts": (1, 256, 1600, 16, 8, 64),
    "wide": (2, 300, 300, 24, 12, 128),
    "wide and odd": (2, 257, 300, 24, 24, 70),
    "narrow": (2, 300, 300, 32, 16, 20),
}


def test_the_unlike_shapes_take_their_paths(fg):
    cut = ["pack", "tiles"]
    for causal in (False, True):
        launches = {p: forward_launches(fg, *s, None, causal) for p, s in UNLIKE.items()}
        assert launches == {"small": ["token"], "large": cut, "large in parts": cut + ["join"], "wide": cut,
                            "wide and odd": cut, "narrow": cut}


def unlike_inputs(path, seed):
    batch, sq, sk, heads, kv_heads, dim = UNLIKE[path]
    return attention_inputs(seed, batch, sq, sk, heads, kv_heads, dim), dict(batch=batch, heads=heads, kv_heads=kv_heads)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e2, 5e2, 4e3, 6e4, 1e6, 1e9, 1e12, 1e20])
@pytest.mark.parametrize("of", ["k", "v", "kv"])
@pytest.mark.parametrize("path", UNLIKE)
def test_a_large_key_or_value_changes_nothing_for_queries_that_do_not_see_it(fg, hip, path, of, size):
    (q, k, v, g), kw = unlike_inputs(path, 70)
    batch, sq, sk = UNLIKE[path][:3]
    at = 3 * sq // 4  # the query that sees it first, and its key
    want = attention_ref.attention(q, k, v, causal=True, g=g, **kw)
    g = g.reshape(batch, sq, -1).copy()
    g[:, at:] = 0  # the others' gradients
    g = g.reshape(batch * sq, -1)
    want_grads = attention_ref.attention(q, k, v, causal=True, g=g, **kw)
    for x, name in ((k, "k"), (v, "v")):
        if name in of:
            x.reshape(batch, sk, -1)[:, at + sk - sq] *= np.float32(size)
    got = run_both(fg, q, k, v, g, causal=True, **kw)
    rows = (np.arange(batch * sq) % sq) < at
    check("y", got["y"][rows], *(x[rows] for x in want["y"]))
    check("dq", got["dq"][rows], *(x[rows] for x in want_grads["dq"]))
    if "k" not in of:  # a large key makes the probabilities of those that see it what they are not here
        keys = (np.arange(batch * sk) % sk) < at + sk - sq
        check("dv", got["dv"][keys], *(x[keys] for x in want_grads["dv"]))
        # Values up to 2^10 apart are cut operands', and dk's ds are cut below
        # 2^-24 once times 2^12 over the powers of two above |g'| (at most |g|)
        # and above the head's largest |v|, each up to twice the norm: 2^-34 |g| |v|
        # a pair, times the largest |q| scale and the pairs of a key.
        value, bound = want_grads["dk"]
        if size < 2.0 ** 10:
            dim, group = UNLIKE[path][5], UNLIKE[path][3] // UNLIKE[path][4]
            norm = lambda x: np.sqrt((x.reshape(-1, dim).astype(np.float64) ** 2).sum(1)).max()  # noqa: E731
            bound = bound + 2.0 ** -34 * norm(g) * norm(v) * np.abs(q).max() * dim ** -0.5 * group * sq
        check("dk", got["dk"][keys], value[keys], bound[keys])


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e2, 5e2, 4e3, 1e6, 1e9, 1e12])
@pytest.mark.parametrize("path", UNLIKE)
def test_a_value_that_weighs_nothing_changes_nothing(fg, hip, path, size):
    # Its key scores -10^4 or less, so that its probability is 0 in float32 and
    # in float64: the call without that key.
    (q, k, v, g), kw = unlike_inputs(path, 71)
    batch, sq, sk, heads, kv_heads, dim = UNLIKE[path]
    q[:, ::dim] = np.abs(q[:, ::dim]) + 0.5
    at = sk // 3
    rest = np.arange(batch * sk) % sk != at
    want = attention_ref.attention(q, k[rest], v[rest], g=g, **kw)
    k.reshape(batch, sk, kv_heads, dim)[:, at, :, 0] = -4e4 * np.sqrt(dim)
    v.reshape(batch, sk, -1)[:, at] *= np.float32(size)
    got = run_both(fg, q, k, v, g, **kw)
    check("y", got["y"], *want["y"])
    check("dq", got["dq"], *want["dq"])
    for name in ("dk", "dv"):
        check(name, got[name][rest], *want[name])
        assert not got[name][~rest].any(), name


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e2, 5e2, 4e3, 6e4, 1e6, 1e9, 1e12])  # either side of what cut operands take
@pytest.mark.parametrize("path", UNLIKE)
def test_columns_beside_a_large_one(fg, hip, path, size):
    # A column of the values that is large in each head, where the gradient is 0:
    # the other columns, and the gradients, are as without it. A column of the
    # keys that is large where the queries are 0, the same.
    (q, k, v, g), kw = unlike_inputs(path, 72)
    batch, sq, sk, heads, kv_heads, dim = UNLIKE[path]
    q[:, 1::dim] = 0
    g[:, ::dim] = 0
    want = attention_ref.attention(q, k, v, g=g, **kw)
    v[:, ::dim] *= np.float32(size)
    k[:, 1::dim] *= np.float32(size)
    got = run_both(fg, q, k, v, g, **kw)
    for name, large in (("y", 0), ("dq", 1), ("dk", None), ("dv", None)):
        columns = np.arange(got[name].shape[1]) % dim != (-1 if large is None else large)
        check(name, got[name][:, columns], *(x[:, columns] for x in want[name]))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e2, 5e2, 4e3, 1e6, 1e9, 1e12])
@pytest.mark.parametrize("of", ["q", "g"])
@pytest.mark.parametrize("path", UNLIKE)
def test_a_large_query_or_gradient_changes_nothing_for_keys_that_it_does_not_see(fg, hip, path, of, size):
    (q, k, v, g), kw = unlike_inputs(path, 73)
    batch, sq, sk = UNLIKE[path][:3]
    at = sq // 3
    want = attention_ref.attention(q, k, v, causal=True, g=g, **kw)
    x = {"q": q, "g": g}[of]
    x.reshape(batch, sq, -1)[:, at] *= np.float32(size)
    got = run_both(fg, q, k, v, g, causal=True, **kw)
    keys = (np.arange(batch * sk) % sk) > at + sk - sq
    rows = (np.arange(batch * sq) % sq) != at
    for name in ("dk", "dv"):
        check(name, got[name][keys], *(x[keys] for x in want[name]))
    for name in ("y", "dq"):
        check(name, got[name][rows], *(x[rows] for x in want[name]))


# The same through every launch of the gradients: both in one, one for each, and
# queries or keys in parts, at every number of column groups.
EVERY = {
    "one launch, 1": (3, 70, 90, 4, 2, 30),
    "one launch, 2": (3, 70, 90, 4, 2, 50),
    "one launch, 3": (3, 70, 90, 4, 2, 80),
    "one launch, 4": (3, 70, 90, 4, 2, 128),
    "parts, 2": (1, 520, 300, 64, 1, 64),
    "parts, 4": (1, 300, 900, 6, 2, 100),
    "two launches, 1": (17, 130, 140, 40, 40, 16),
    "two launches, 2": (16, 130, 130, 24, 24, 50),
    "two launches, 3": (16, 130, 130, 20, 20, 70),
    "two launches, 4": (16, 130, 130, 20, 20, 110),
}


def test_the_shapes_reach_every_launch_of_the_gradients(fg):
    names = set()
    for batch, sq, sk, heads, kv_heads, dim in EVERY.values():
        q, k = lazy(fg, batch * sq, heads * dim), fg.Tensor.zeros([batch * sk, kv_heads * dim], "hip")
        g = q.attention(k, k, heads=heads, kv_heads=kv_heads, batch=batch, causal=True).sum([0, 1]).gradient([q])[0]
        for it in fg.debug_plan([g], fuse=True, render_hip=True)["items"]:
            names |= {l["name"] for l in it["launches"]} if it["class"] == "attention_grad" else set()
    want = {f"fg_attention_{n}_{i}" for n in ("grad_pack", "grads", "grad_kv", "grad_q") for i in (1, 2, 3, 4)}
    assert want <= names and {"fg_attention_grad_sum_2", "fg_attention_grad_sum_4"} <= names, want - names


@pytest.mark.gpu
@pytest.mark.parametrize("path", EVERY)
def test_operands_of_unlike_sizes_in_every_launch(fg, hip, path, monkeypatch):
    monkeypatch.setitem(UNLIKE, path, EVERY[path])
    for of in ("v", "kv"):
        test_a_large_key_or_value_changes_nothing_for_queries_that_do_not_see_it(fg, hip, path, of, 1e9)
    for of in ("q", "g"):
        test_a_large_query_or_gradient_changes_nothing_for_keys_that_it_does_not_see(fg, hip, path, of, 1e9)
    test_a_value_that_weighs_nothing_changes_nothing(fg, hip, path, 1e9)
    test_columns_beside_a_large_one(fg, hip, path, 1e9)


@pytest.mark.gpu
@pytest.mark.parametrize("path", UNLIKE)
def test_gradients_that_grow_over_the_sequence(fg, hip, path):
    # Blocks of queries 2^12 apart, 2^50 and more in all: the last keys are seen
    # by the last, smallest gradients only.
    (q, k, v, g), kw = unlike_inputs(path, 74)
    batch, sq, sk = UNLIKE[path][:3]
    g = g.reshape(batch, sq, -1)
    want = attention_ref.attention(q, k, v, causal=True, g=g.reshape(batch * sq, -1), **kw)
    scale = 2.0 ** (12 * ((sq - 1 - np.arange(sq)) // 32))
    g = (g * scale[:, None].astype(np.float32)).reshape(batch * sq, -1)
    got = run_both(fg, q, k, v, g, causal=True, **kw)
    rows = np.tile(scale[:, None], (batch, 1))
    check("dq", got["dq"] / rows, *want["dq"])
    last = (np.arange(batch * sq) % sq) >= sq - sq % 32 if sq % 32 else (np.arange(batch * sq) % sq) >= sq - 32
    keys = (np.arange(batch * sk) % sk) >= sk - last[:sq].sum()
    for name in ("dk", "dv"):
        check(name, got[name][keys], *(x[keys] for x in want[name]))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [1, 3, 63, 127])
@pytest.mark.parametrize("sk", [1300, 2000])
def test_one_token_of_an_odd_head_in_an_odd_number_of_parts(fg, hip, dim, sk):
    # The parts' sums are an odd number of floats.
    q, k, v, _ = attention_inputs(80 + dim, 1, 1, sk, 1, 1, dim)
    want = attention_ref.attention(q, k, v, 1, 1, 1)
    check("y", new(fg, q).attention(new(fg, k), new(fg, v), heads=1).numpy(), *want["y"])


# ── the largest sizes ───────────────────────────────────────────────────────


def test_more_rows_than_the_kernels_count_are_refused(fg):
    # Nothing of these sizes is allocated: a call past its limit is refused before.
    z = lambda *s: fg.Tensor.zeros(list(s), "hip")  # noqa: E731
    for heads in ((1 << 31) - 1, (1 << 31) - 1024):
        with pytest.raises(fg.FerrogradError, match="heads of tokens"):
            z(1, 2 * heads).norm_rotate(z(2), fg.Tensor.zeros([1], "hip", fg.I32), heads=heads)
    k = z(5, 1)
    with pytest.raises(fg.FerrogradError, match="share a key head"):
        z(1 << 28, 8).attention(k, k, heads=8, kv_heads=1)
    z(1 << 27, 8).attention(k, k, heads=8, kv_heads=1)


def test_more_threads_than_a_launch_takes_are_refused(fg):
    plan = lambda t: fg.debug_plan([t], fuse=True, render_hip=True)  # noqa: E731
    n = (1 << 34) - 512  # 512 elements a workgroup of 128
    assert plan(fg.Tensor.zeros([n], "hip").dropout(0.5, 1))["items"][0]["launches"][0]["grid"] == (1 << 25) - 1
    with pytest.raises(fg.FerrogradError, match="threads in one launch"):
        plan(fg.Tensor.zeros([n + 1], "hip").dropout(0.5, 1))
    q = fg.Tensor.zeros([1 << 23, 8], "hip").with_requires_grad(True)  # 2^23 sequences of one token: 2^25 blocks to cut
    y = q.attention(q, q, heads=1, batch=1 << 23)
    plan(y)
    with pytest.raises(fg.FerrogradError, match="threads in one launch"):
        plan(y.sum([0, 1]).gradient([q])[0])


def test_an_eps_that_float32_does_not_hold_is_refused(fg):
    x, w, pos = lazy(fg, 6, 8), lazy(fg, 4), lazy(fg, 6, dtype=fg.I32)
    for eps in (1e39, 1e-50, float("inf"), float("nan"), -1e-9):
        with pytest.raises(fg.FerrogradError, match="eps"):
            x.norm_rotate(w, pos, heads=2, eps=eps)
    for eps in (0.0, 1e-40, 3e38):
        x.norm_rotate(w, pos, heads=2, eps=eps)


@pytest.mark.parametrize("kw", [dict(heads=0), dict(heads=-2), dict(heads=2, kv_heads=0), dict(heads=2, kv_heads=-2),
                                dict(heads=2, head_dim=0)])
def test_a_layer_of_no_heads_is_refused(fg, kw):
    from ferrograd_amd.attention import SelfAttention

    with pytest.raises(fg.FerrogradError, match="SelfAttention"):
        SelfAttention(32, device="hip", **kw)


# ── the workspace ───────────────────────────────────────────────────────────


@pytest.mark.gpu
def test_cleared_caches_give_the_workspace_back(fg, hip):
    import gc

    import torch

    from ferrograd_amd.hip import Context, api, check as hip_check

    ctx = Context.of_device()
    q = fg.Tensor.zeros([4096, 16 * 64], "hip").with_requires_grad(True)
    x = new(fg, seeded(90).standard_normal((4096, 16 * 64)).astype(np.float32))

    def gradient():
        return q.add(x).attention(x, x, heads=16, causal=True).sum([0, 1]).gradient([q])[0]

    workspace = max(it.get("workspace", 0) for it in fg.debug_plan([gradient()], fuse=True, render_hip=True)["items"])
    assert workspace > 1 << 26

    def free():
        gc.collect()
        hip_check(api().fg_hip_trim(ctx.h))
        return torch.cuda.mem_get_info()[0]

    first = gradient().numpy()
    held = free()
    fg.clear_caches()
    cleared = free()
    assert cleared - held >= workspace * 9 // 10, (held, cleared, workspace)
    assert np.array_equal(gradient().numpy(), first)  # and it is taken again


# ── layers, trained ─────────────────────────────────────────────────────────


@pytest.mark.gpu
def test_a_sequence_classifier_has_the_loss_and_the_updates_of_its_parameters(fg, hip):
    import torch

    from ferrograd_amd.attention import SelfAttention
    from test_operators import Torch64, philox

    features, heads, kv_heads, batch, n, classes, lr = 32, 4, 2, 4, 20, 5, 0.25
    fg.reset_init_seed(6)
    layers = [SelfAttention(features, heads, kv_heads, device=hip, dropout=0.125, seed=i) for i in range(2)]
    head = fg.Linear(features, classes, hip)
    params = [p for l in layers for p in l.parameters()] + head.parameters()
    opt = fg.Sgd(params, lr)
    r = seeded(91)
    pos = np.tile(np.arange(n, dtype=np.int32), batch)
    lengths = np.array([20, 7, 13, 1], np.int32)
    tp, tl = new(fg, pos), new(fg, lengths)
    # Each layer's values are off by at most 9 * 16 half steps times the terms
    # summed over (as for one layer's), and there are two and the classifier.
    tol = 3 * 9 * 16 * (2 * features + n + batch * n) * U
    for step in range(3):
        xs = r.standard_normal((batch * n, features)).astype(np.float32)
        ts = np.eye(classes, dtype=np.float32)[r.integers(0, classes, batch * n)]
        before = [p.numpy().astype(np.float64) for p in params]
        h = new(fg, xs)
        for l in layers:
            h = h.add(l(h, tp, batch, tl))
        loss = head(h).cross_entropy(new(fg, ts))
        opt.zero_grad()
        loss.backward()
        opt.step()
        got = float(loss.to_vec()[0])
        ps = [torch.tensor(p, requires_grad=True) for p in before]
        z, at = torch.tensor(xs.astype(np.float64)), 0
        for i in range(2):
            wq, wk, wv, wo, nq, nk = ps[at:at + 6]
            at += 6
            q = Torch64.norm_rotate(z @ wq.T, nq, torch.tensor(pos), heads, 1e-6, 10000.0)
            k = Torch64.norm_rotate(z @ wk.T, nk, torch.tensor(pos), kv_heads, 1e-6, 10000.0)
            out = Torch64.attention(q, k, z @ wv.T, heads, kv_heads, batch, torch.tensor(lengths)) @ wo.T
            keep = philox(out.numel(), i, step).reshape(out.shape) >= 1 << 29
            z = z + out * torch.tensor(keep / 0.875)
        want = -(torch.log_softmax(z @ ps[at].T + ps[at + 1], 1) * torch.tensor(ts.astype(np.float64))).sum() / (batch * n)
        assert abs(got - float(want.detach())) <= tol * abs(float(want.detach())), (step, got, float(want.detach()))
        for i, (p, b, g) in enumerate(zip(params, before, torch.autograd.grad(want, ps))):
            update, g = (b - p.numpy()) / lr, g.numpy()
            rounding = U * np.linalg.norm(b) / lr  # of the updated parameter
            assert np.linalg.norm(update - g) <= tol * np.linalg.norm(g) + 2 * rounding, (step, i)
