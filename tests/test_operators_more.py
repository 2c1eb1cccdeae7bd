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
