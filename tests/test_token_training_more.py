"""Embedding, layer norm, the loss of token labels and clipping, further: how
Python reaches them, and each of their kernels against float64."""
import inspect

import numpy as np
import pytest


# ── from Python (no GPU) ────────────────────────────────────────────────────


def test_tensors_are_given_by_position_or_by_name(fg, cpu):
    a = fg.Tensor.new(np.arange(6, dtype=np.float32), [2, 3], "cpu").with_requires_grad(True)
    loss = a.mul(a).sum([0, 1])
    for got in (loss.gradient([a]), loss.gradient(targets=[a]), loss.gradient((a,)), fg.Tensor.gradient(loss, targets=[a])):
        assert np.array_equal(got[0].numpy(), 2 * a.numpy())
    for call in (lambda ts: fg.Tensor.realize_many(ts), lambda ts: fg.Tensor.realize_many(tensors=ts), lambda ts: a.realize_many(tensors=ts)):
        b, c = a.add(a), a.neg()
        call([b, c])
        assert b.is_realized() and c.is_realized()
    assert list(inspect.signature(loss.gradient).parameters) == ["targets"]
    assert list(inspect.signature(fg.Tensor.realize_many).parameters) == ["tensors"]
    for bad in (loss.gradient, fg.Tensor.realize_many):
        for args, kw in (((), {}), (([a], [a]), {}), ((), dict(other=[a])), (([a],), dict(targets=[a])), (([a],), dict(tensors=[a]))):
            with pytest.raises(TypeError):
                bad(*args, **kw)
