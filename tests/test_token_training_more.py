"""Embedding, layer norm, the loss of token labels and clipping, further: how
Python reaches them, and each of their kernels against float64."""
import inspect
import os
import subprocess
import sys
import threading
import time

import numpy as np
import pytest

from conftest import graphs_on, seeded
from test_token_training import U, check, layer_norm64, loss64, new, normal, some_ids, weighted


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


def test_a_train_step_tells_labels_by_their_shape(fg, cpu):
    # One number a row is a label. Rows of numbers are cross_entropy's targets, of whichever type, as before there were labels.
    from ferrograd_amd.mlp import Mlp, train_step

    x, rows = fg.Tensor.new(seeded(4).standard_normal((2, 3)).astype(np.float32), [2, 3], "cpu"), np.eye(4)[[1, 3]]
    for targets in (rows.astype(np.float32), rows.astype(np.int32)):
        t, got = fg.Tensor.new(targets, [2, 4], "cpu"), []
        for step in (train_step, lambda m, opt, x, t: m.forward_preactivations(x)[-1].cross_entropy(t)):
            fg.reset_init_seed(5)
            model = Mlp((3, 4), cpu)
            params = model.parameters()
            opt = fg.Sgd(params, 0.1)
            loss = step(model, opt, x, t)
            if step is not train_step:
                loss.backward()
                opt.step()
            got.append([loss.numpy()] + [p.numpy() for p in params])
        assert all(np.array_equal(a, b) for a, b in zip(*got))
    with pytest.raises(fg.FerrogradError, match=r"target shape \[2, 3\] must match logits shape \[2, 4\]"):
        train_step(model, opt, x, fg.Tensor.new(np.zeros((2, 3), np.int32), [2, 3], "cpu"))
    with pytest.raises(fg.FerrogradError, match="token_cross_entropy: the labels must be i32"):
        train_step(model, opt, x, fg.Tensor.new(np.zeros(2, np.float32), [2], "cpu"))


def test_layer_norm_gradients_of_too_many_columns_are_refused(fg):
    # Forward it is planned; the launch that adds up the weight's gradient would have 2^32 threads.
    x, w = fg.Tensor.zeros([1, 1 << 26], "hip"), fg.Tensor.zeros([1 << 26], "hip").with_requires_grad(True)
    y = x.layer_norm(w)
    fg.debug_plan([y], fuse=True, render_hip=True)
    with pytest.raises(fg.FerrogradError, match=r"layer_norm: .* in one launch, which takes 2\^32 - 1 threads"):
        fg.debug_plan(y.sum([0, 1]).gradient([w]), fuse=True, render_hip=True)


def while_it_runs(call, meanwhile):
    """Seconds that call() took, and how often another thread ran meanwhile, once a millisecond."""
    ticks, go, stop = [], threading.Event(), threading.Event()

    def tick():
        go.set()
        while not stop.wait(0.001):
            meanwhile()
            ticks.append(time.perf_counter())

    thread = threading.Thread(target=tick)
    thread.start()
    go.wait()
    begin = time.perf_counter()
    call()
    end = time.perf_counter()
    stop.set()
    thread.join()
    # Not those next to its ends, where the interpreter itself hands over.
    inside = [t for t in ticks if begin + 0.1 * (end - begin) < t < end - 0.1 * (end - begin)]
    return end - begin, len(inside)


def long_call(fg, kind, size):
    """A call of a time that grows with `size`, and a list of tensors that it was given."""
    a = fg.Tensor.new(np.ones(1 << 12, np.float32), [1 << 12], "cpu").with_requires_grad(True)
    if kind == "realize_many":
        ts = [fg.Tensor.new(np.full(1 << size, i + 1.0, np.float32), [1 << size], "cpu").sqrt().exp().log().sum([0]) for i in range(2)]
        return ts, lambda: fg.Tensor.realize_many(ts)
    y = a
    for _ in range(1 << (size - 10)):
        y = y.mul(a)
    loss, ts = y.sum([0]), [a]
    return ts, lambda: loss.gradient(ts)


@pytest.mark.parametrize("kind", ["realize_many", "gradient"])
def test_other_threads_run_while_the_library_works(fg, cpu, kind):
    for size in range(20, 26):
        # The other thread empties the list, which alone has the tensors: the call keeps them.
        ts, call = long_call(fg, kind, size)
        seconds, ticks = while_it_runs(call, ts.clear)
        if seconds > 0.08:
            break
    assert seconds > 0.08 and ticks >= 3, (seconds, ticks)


BESIDE = """
import sys, threading
sys.path.insert(0, sys.argv[1])
import numpy as np
import ferrograd_amd as fg, oracle
oracle.load()
stop = threading.Event()

def beside():
    while not stop.is_set():
        ts = [fg.Tensor.new(np.ones(64, np.float32), [64], "cpu") for _ in range(20)]
        y = ts[0]
        for t in ts:
            y = y.add(t)
        del ts, y, t

thread = threading.Thread(target=beside)
thread.start()
try:
    a = fg.Tensor.new(np.arange(64, dtype=np.float32) / 64, [64], "cpu").with_requires_grad(True)
    for i in range(200):
        y = a
        for _ in range(30):
            y = y.mul(a).add(a)
        z = a.mul(a).add(a)
        g = y.sum([0]).gradient([a])[0]
        fg.Tensor.realize_many([z])
        assert np.array_equal(z.numpy(), a.numpy() * a.numpy() + a.numpy())
finally:
    stop.set()
    thread.join()
print("done")
"""


def test_tensors_are_made_and_dropped_while_the_library_works(fg, cpu):
    # What collecting garbage does in any thread: a program of its own, which a race would end.
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", BESIDE, root], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout.strip() == "done", (p.returncode, p.stderr[-2000:])


# ── embedding (GPU) ─────────────────────────────────────────────────────────


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim", [(600001, 132), (1100001, 68), (4200001, 5)])
def test_embedding_gradient_of_a_frequent_id_adds_up(fg, hip, tokens, dim):
    # The rows of one id are alike, so that the roundings of a long sum all go one way. A sum of 64 rows has 63
    # additions in float32; all else is in 64 bits, but for the rounding of a chunk's part and of the result.
    row = (1 + np.arange(dim) / dim).astype(np.float32)[None]
    g = new(fg, row).embedding(new(fg, np.zeros(tokens, np.int32))).realize()
    r = np.random.default_rng(310)
    ids = np.where(r.random(tokens) < 0.9, 3, r.integers(0, 7, tokens)).astype(np.int32)
    w = fg.Tensor.zeros([7, dim], "hip").with_requires_grad(True)
    dw = w.embedding(new(fg, ids)).mul(g).sum([0, 1]).gradient([w])[0].numpy()
    want = np.bincount(ids, minlength=7)[:, None] * row.astype(np.float64)
    check("dw", dw, want, 66 * U * want)


# ── clipping (GPU) ──────────────────────────────────────────────────────────


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [1e-6, 1e-9, 1e-12, 1e-20, 1e-36, 1e-43, 1e-60])
def test_clip_norm_by_factors_below_the_normal_range(fg, hip, max_norm):
    # Norms of about 1e33 and more: factors of 1e-39 and less, of products that are numbers of full precision.
    xs = [(normal(300 + i, n) * 1e31).astype(np.float32) for i, n in enumerate((4096, 5001, 3))]
    norm = np.sqrt(sum((x.astype(np.float64) ** 2).sum() for x in xs))
    got, clipped = fg.clip_norm([new(fg, x) for x in xs], max_norm)
    fg.Tensor.realize_many([got] + clipped)
    check("norm", got.numpy(), np.array([norm]), 1.01 * U * norm)
    step = 2.0 ** -149  # of numbers below the normal range
    for x, y in zip(xs, clipped):
        want = x.astype(np.float64) * (max_norm / norm)
        # The factor's digits are rounded once and the product once, and where it is below the normal range once more.
        assert np.all(np.abs(y.numpy() - want) <= 2.01 * U * np.abs(want) + 0.51 * step), max_norm


# ── every kernel, over many rows (GPU) ──────────────────────────────────────
#
# Rows are of a few different ones, so that float64 has these alone to make, and
# equal rows have to come out equal in every bit wherever they are (where no note
# says otherwise). Sums over all
# rows are of small whole numbers, of which every partial sum is exact, where they
# can be. Each width goes through its kernel twice: with more rows than one round
# of workgroups takes, and with outputs of 64 MB, which go past the caches.

KINDS = 61  # of rows
STREAM = 1 << 24  # floats of an output past the caches


def drawn(seed, rows):
    """Which of the kinds of rows each row is, every kind among them, and how many there are of each."""
    which = seeded(seed).integers(0, KINDS, rows)
    which[:KINDS] = np.arange(KINDS)[:rows]
    return which, np.bincount(which, minlength=KINDS)


def whole_numbers(seed, *shape):
    return seeded(seed).integers(-2, 3, shape).astype(np.float32)


def check_kinds(name, got, which, want, bound, alike=True):
    """Rows against those of their kind; equal rows are alike, or else each is within the bound."""
    if alike:
        assert np.array_equal(got, got[:KINDS][which]), name
        check(name, got[:KINDS], want, bound)
    else:
        check(name, got, want[which], bound[which])


WIDTHS = [  # whole and broken vectors of every split of a row over lanes
    8, 32, 3, 27, 64, 51, 128, 117, 256, 203, 512, 473, 1024, 1001, 2048, 1999, 4096, 4001, 8192, 8155, 16384, 16001, 32768, 32003,
]


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [1, 3, 4, 27, 64, 51, 128, 117, 256, 203, 1028])
@pytest.mark.parametrize("kind", ["words", "padded", "one"])
@pytest.mark.parametrize("many", [False, True])
def test_embedding_and_its_gradient_are_exact(fg, hip, dim, kind, many):
    tokens, vocab = STREAM // dim + 3 if many else 70001, 2999
    r = seeded(320)
    ids = some_ids("words" if kind == "padded" else kind, tokens, vocab, 321)
    if kind == "padded":
        ids[r.random(tokens) < 1 / 3] = 5
        ids[r.random(tokens) < 0.1] = -1
    w, table = whole_numbers(322, vocab, dim), whole_numbers(323, KINDS, dim)
    which = r.integers(0, KINDS, tokens)
    tw = new(fg, w, True)
    y, dw = weighted(fg, tw.embedding(new(fg, ids), 0.5), table[which], [tw])
    inside = ids >= 0
    assert np.array_equal(y, np.where(inside[:, None], 0.5 * w[ids], 0.0))
    # Of each id, how many tokens have each kind of gradient. All sums are below 2^24.
    counts = np.bincount(ids[inside] * KINDS + which[inside], minlength=vocab * KINDS).reshape(vocab, KINDS)
    assert np.array_equal(dw, 0.5 * (counts @ table.astype(np.float64)))


def norm_splits(rows, dim):
    """Rows that a lane sums the weights' gradients of, and the additions that its sums go through after it: the rows of
    a workgroup, of a slice of the workgroups, and of the slices."""
    lanes = next((l for l, k in ((8, 1), (16, 1), (32, 1), (64, 4), (256, 4), (512, 4), (1024, 4)) if 4 * l * k >= dim), None)
    if lanes is None:
        return -(-rows // min(rows, 32)), 6
    threads = max(256, lanes)
    groups = threads // lanes
    blocks = min(-(-rows // groups), 4 * 256 * 256 // threads)
    return -(-rows // (groups * blocks)), groups + -(-blocks // 32) + 5


def norm_rows(rows, dim):
    if rows == "many":
        return STREAM // dim + 3
    lanes = max(8, 1 << max(0, (dim - 1).bit_length() - 2)) if dim <= 256 else 64 if dim <= 1024 else 256
    # More than two rounds of the gradient's workgroups, the last one not full.
    return min(2 * 1024 * 256 // lanes + 77, STREAM // dim - 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", WIDTHS + [40001])
@pytest.mark.parametrize("rows", ["some", "many"])
def test_layer_norm_of_all_widths_over_many_rows(fg, hip, dim, rows):
    n = norm_rows(rows, dim)
    x, g, w = 2 + 3 * normal(330, KINDS, dim), whole_numbers(331, KINDS, dim), 1 + 0.1 * normal(332, dim)
    b = 0.1 * normal(333, dim)
    which, counts = drawn(334, n)
    tx, tw, tb = new(fg, x[which], True), new(fg, w, True), new(fg, b, True)
    y, dx, dw, db = weighted(fg, tx.layer_norm(tw, tb), g[which], [tx, tw, tb])
    (wy, ey), (wx, ex), *_ = layer_norm64(x, w, b, g, 1e-5)
    check_kinds("y", y, which, wy, ey)
    check_kinds("dx", dx, which, wx, ex)
    assert np.array_equal(db, counts @ g.astype(np.float64))  # below 2^24
    # dw: each row's term with its bound, and the additions of a lane's rows and after them.
    want, bound, size = np.zeros(dim), np.zeros(dim), np.zeros(dim)
    for i in np.flatnonzero(counts):
        _, _, (term, off), _ = layer_norm64(x[i:i + 1], w, b, g[i:i + 1], 1e-5)
        want += counts[i] * term
        bound += counts[i] * off
        size += counts[i] * np.abs(term)
    lane, after = norm_splits(n, dim)
    check("dw", dw, want, bound + 1.01 * (lane + after) * U * size)
    # Without a bias, and forward alone.
    assert np.array_equal(tx.layer_norm(tw, tb).numpy(), y)
    y, dx, dw2 = weighted(fg, tx.layer_norm(tw), g[which], [tx, tw])
    (wy, ey), (wx, ex), *_ = layer_norm64(x, w, None, g, 1e-5)
    check_kinds("y", y, which, wy, ey)
    check_kinds("dx", dx, which, wx, ex)
    assert np.array_equal(dw2, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 31, 33, 67, 100])
@pytest.mark.parametrize("dim", [20000, 40001])
def test_layer_norm_weights_of_parts_of_the_rows(fg, hip, rows, dim):
    # Rows in up to 32 parts of equal length, of which the last ones may have none.
    g, x = whole_numbers(340, rows, dim), normal(341, rows, dim)
    tx, tw, tb = new(fg, x, True), new(fg, 1 + 0.1 * normal(342, dim), True), new(fg, normal(343, dim), True)
    y, dx, dw, db = weighted(fg, tx.layer_norm(tw, tb), g, [tx, tw, tb])
    assert np.array_equal(db, g.astype(np.float64).sum(0))
    for name, a, (want, bound) in zip(("y", "dx", "dw"), (y, dx, dw), layer_norm64(x, tw.numpy(), tb.numpy(), g, 1e-5)):
        check(name, a, want, bound)


LOSS_WIDTHS = WIDTHS + [65536, 65003, 70000, 70003]


@pytest.mark.gpu
@pytest.mark.parametrize("classes", LOSS_WIDTHS)
@pytest.mark.parametrize("many", [False, True])
def test_token_cross_entropy_of_all_widths_over_many_rows(fg, hip, classes, many):
    # Short rows: more than a round of workgroups, of two rows each and more. Long ones are one a workgroup.
    n = STREAM // classes + 3 if many else min(70001, STREAM // classes - 1)
    r = seeded(350)
    x, labels = 3 * normal(351, KINDS, classes), r.integers(0, classes, KINDS).astype(np.int32)
    x[r.random(x.shape) < 0.1] = -np.inf
    x[np.arange(KINDS), labels] = r.standard_normal(KINDS)
    labels[r.random(KINDS) < 0.3] = -1
    labels[7] = classes
    which, counts = drawn(352, n)
    total = counts[(labels >= 0) & (labels < classes)].sum()
    tx, tl = new(fg, x[which], True), new(fg, labels[which])
    loss = tx.token_cross_entropy(tl)
    dx = loss.gradient([tx])[0]
    fg.Tensor.realize_many([loss, dx])
    want, bound = 0.0, 0.0
    for i in np.flatnonzero(counts):
        (each, off), _ = loss64(x[i:i + 1], labels[i:i + 1])
        want, bound = want + counts[i] * each / total, bound + counts[i] * off / total
    # The rows of a workgroup are rounded once, and the mean.
    check("loss", loss.numpy(), want, bound + 2 * U * want)
    valid = ((labels >= 0) & (labels < classes)).sum()
    # Long rows of broken vectors are read from the cache line that they begin in: sums of equal rows that begin
    # elsewhere in theirs are of other numbers, and as good.
    alike = classes % 4 == 0 or classes <= 4096
    check_kinds("dx", dx.numpy(), which, *loss64(x, labels, valid / total)[1], alike)
    # Alone, and under a gradient that is not 1.
    assert np.array_equal(tx.token_cross_entropy(tl).numpy(), loss.numpy())
    scaled = tx.token_cross_entropy(tl).mul(new(fg, np.array([-2.5], np.float32))).gradient([tx])[0].numpy()
    check_kinds("scaled", scaled, which, *loss64(x, labels, -2.5 * valid / total)[1], alike)


@pytest.mark.gpu
def test_a_norm_past_the_range_clips_as_itself(fg, hip):
    x = np.where(normal(305, 5001) > 0, 3e38, -2e38).astype(np.float32)
    total = np.sqrt((x.astype(np.float64) ** 2).sum())  # 2e40
    for max_norm in (1.0, 1e39):
        norm, (y,) = fg.clip_norm([new(fg, x)], max_norm)
        fg.Tensor.realize_many([norm, y])
        assert norm.numpy()[0] == np.inf
        want = x.astype(np.float64) * (max_norm / total)
        check("clipped", y.numpy(), want, 2.01 * U * np.abs(want))


@pytest.mark.gpu
@pytest.mark.parametrize("count", [3, 20, 70])
def test_clip_norm_of_more_than_the_caches_hold(fg, hip, count):
    # Squares of whole numbers: the norm is rounded once. Products past the caches, squares of the first chunks too.
    r = seeded(360)
    pattern = whole_numbers(361, 1 << 20)
    xs = [np.resize(np.roll(pattern, 1000 * i), 2 * STREAM // count + int(r.integers(9000))) for i in range(count)]
    total = np.sqrt(sum(float((x.astype(np.float64) ** 2).sum()) for x in xs))
    norm, clipped = fg.clip_norm([new(fg, x) for x in xs], 1.0)
    fg.Tensor.realize_many([norm] + clipped)
    check("norm", norm.numpy(), np.array([total]), 1.01 * U * total)
    for x, y in zip(xs, clipped):
        for value in range(-2, 3):  # a number's products are all the same
            got = np.unique(y.numpy()[x == value])
            assert len(got) == 1 and abs(float(got[0]) - value / total) <= 2.01 * U * abs(value / total)


# ── calls together (GPU) ────────────────────────────────────────────────────


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_replayed_steps_read_the_batches_that_they_narrow_to(fg, hip, graphs):
    # The batch's start changes from step to step, under one plan: ids, labels and rows added to them.
    rows, batch, vocab, dim = 96, 16, 19, 12
    r = seeded(370)
    ids, labels = (r.integers(-1, vocab, rows).astype(np.int32) for _ in range(2))
    more, w, n = normal(371, rows, dim), normal(372, vocab, dim), normal(373, dim)
    tids, tlabels, tmore, tw, tn = new(fg, ids), new(fg, labels), new(fg, more), new(fg, w, True), new(fg, n, True)

    def step(ids, labels, more):
        x = tw.embedding(ids, 2.0).add(more).layer_norm(tn)
        loss = x.matmul(tw.permute([1, 0])).token_cross_entropy(labels)
        norm, clipped = fg.clip_norm(loss.gradient([tw, tn]), 0.01)
        outs = [loss, norm] + clipped
        fg.Tensor.realize_many(outs)
        new(fg, normal(60, 1000)).exp().numpy()  # other work in between
        return [t.numpy() for t in outs]

    starts = [0, 5, 16, 80, 5, 33, 79, 0]
    fresh = [step(*(new(fg, a[s:s + batch]) for a in (ids, labels, more))) for s in starts]
    with graphs_on(fg, 2 if graphs else 0):
        fg.clear_caches()
        for s, want in list(zip(starts, fresh)) * 2:
            got = step(*(t.narrow(0, s, batch) for t in (tids, tlabels, tmore)))
            assert all(np.array_equal(a, b) for a, b in zip(got, want)), s


@pytest.mark.gpu
def test_losses_of_the_same_logits_add_up(fg, hip):
    # Two labels a row, and the same ones twice: each loss is made beside its gradient.
    x, l0, l1 = 3 * normal(380, 33, 50), *(seeded(381 + i).integers(-1, 50, 33).astype(np.int32) for i in range(2))
    tx = new(fg, x, True)
    losses = [tx.token_cross_entropy(new(fg, l)) for l in (l0, l1, l0)]
    total = losses[0].add(losses[1]).add(losses[2])
    dx = total.gradient([tx])[0]
    fg.Tensor.realize_many([total, dx])
    ((a, ea), (da, eda)), ((b, eb), (db, edb)) = loss64(x, l0), loss64(x, l1)
    check("total", total.numpy(), 2 * a + b, 2 * ea + eb + 3 * U * (2 * a + b))
    check("dx", dx.numpy(), 2 * da + db, 2 * eda + edb + 3 * U * (2 * np.abs(da) + np.abs(db)))
    check("loss", losses[1].numpy(), b, eb)


@pytest.mark.gpu
def test_micro_batches_add_up_before_they_are_clipped(fg, hip):
    w, g = normal(390, 11, 8), normal(391, 2, 20, 8)
    ids = seeded(392).integers(0, 11, (2, 20)).astype(np.int32)
    tw = new(fg, w, True)
    opt = fg.Sgd([tw], 0.25)
    for i in range(2):
        tw.embedding(new(fg, ids[i])).mul(new(fg, g[i])).sum([0, 1]).backward()
    norm = opt.clip_grad_norm(0.5)
    opt.step()
    dw, size = np.zeros(w.shape), np.zeros(w.shape)
    for i in range(2):
        np.add.at(dw, ids[i], g[i])
        np.add.at(size, ids[i], np.abs(g[i]))
    total = np.sqrt((dw ** 2).sum())
    # Sums of at most 20 rows in each half, and their sum; the norm and the products by roundings of these.
    off = 21 * U * size
    part = np.sqrt((off ** 2).sum())
    check("norm", norm.numpy(), np.array([total]), part + U * total)
    want = w - 0.25 * dw * (0.5 / total)
    check("step", tw.numpy(), want, 0.25 * (0.5 / total) * (off + np.abs(dw) * (part / total + 4 * U)) + U * np.abs(want))
    assert total > 0.5
