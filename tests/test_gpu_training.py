"""Dropout, layer norm for training and the gated recurrence, forward and backward, against
plain implementations in 64 bits.

Dropout is compared bit for bit. The others carry bounds that follow from the formulas:
u = 2^-24 is half an ulp, a sum of n terms whose chains of additions are at most k long is off
by at most k u times the sum of the terms' magnitudes, and each further rounding adds u of its
result. Every bound is computed from the 64-bit values of the case it is used for.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24


def dev(a, shift=0):
    """The array on the GPU; shift = 1..3 starts it that many elements into an allocation (not
    16-byte aligned)."""
    t = torch.from_numpy(np.ascontiguousarray(a))
    if not shift:
        return t.cuda()
    buf = torch.zeros(t.numel() + shift, dtype=t.dtype, device="cuda")
    buf[shift:] = t.reshape(-1).cuda()
    return buf[shift:].view(t.shape)


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def within(got, want, bound, what):
    got, want, bound = (np.asarray(v, np.float64) for v in (got, want, bound))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = np.abs(got - want)
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], off[bad][:4],
                           np.broadcast_to(bound, off.shape)[bad][:4])


def keep_of(oracle, shape, p, seed, offset):
    n = math.prod(shape)
    return oracle.random("uniform", n, seed, offset, 0.0, 1.0).astype(np.float64).reshape(shape) >= p


def scale_of(p):
    return np.float32(1 / (1 - p)) if p < 1 else np.float32(0)


# ------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("count,shift,offset", [(0, 0, 0), (1, 0, 0), (1, 1, 3), (3, 0, 2), (4, 0, 0), (5, 2, 1),
                                                (1023, 0, 0), (1024, 0, 5), (4099, 3, 6), (100003, 0, 0),
                                                (1 << 20, 0, (1 << 32) - 2), ((1 << 20) + 1, 1, (1 << 34) + 3)])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_is_the_stream_s_mask(tcx, oracle, count, shift, offset, residual):
    rng = np.random.default_rng(count)
    x = rng.normal(size=count).astype(np.float32)
    r = rng.normal(size=count).astype(np.float32) if residual else None
    p, seed = 0.3, 2**63 + 12345
    got = host(tcx.dropout(dev(x, shift), p, seed, offset=offset, residual=None if r is None else dev(r, shift)))
    want = np.where(keep_of(oracle, x.shape, p, seed, offset), x * scale_of(p), np.float32(0)) if count else x
    if residual:
        want = r + want
    assert got.dtype == np.float32 and got.tobytes() == want.astype(np.float32).tobytes()


@pytest.mark.parametrize("p", [0, 0.0, 1e-9, 2.0**-24, 0.1, 0.5, 0.999999, 1.0 - 2.0**-24, 1, 1.0])
def test_dropout_probabilities(tcx, oracle, p):
    x = np.random.default_rng(3).normal(size=(37, 211)).astype(np.float32)
    got = host(tcx.dropout(dev(x), p, 7))
    want = np.where(keep_of(oracle, x.shape, p, 7, 0), x * scale_of(p), np.float32(0))
    assert got.tobytes() == want.astype(np.float32).tobytes()
    if p == 0:
        assert got.tobytes() == x.tobytes()
    if p == 1:
        assert not got.any()


def test_dropout_leaves_nothing_of_what_it_drops(tcx, oracle):
    keep = keep_of(oracle, (64, 100), 0.4, 11, 9)
    for bad in (np.nan, np.inf, -np.inf):
        x = np.where(keep, np.float32(1.5), np.float32(bad)).astype(np.float32)
        got = host(tcx.dropout(dev(x), 0.4, 11, offset=9, residual=dev(np.ones_like(x))))
        assert np.isfinite(got).all()
        assert (got[~keep] == 1).all()
    x = np.where(keep, np.float32(np.nan), np.float32(1)).astype(np.float32)
    got = host(tcx.dropout(dev(x), 0.4, 11, offset=9))
    assert np.isnan(got[keep]).all() and not got[~keep].any()


def test_dropout_backward_is_the_gradient(tcx, oracle):
    rng = np.random.default_rng(5)
    x, dy, v = (rng.normal(size=(23, 77)) for _ in range(3))
    keep = keep_of(oracle, x.shape, 0.2, 99, 13)
    got = host(tcx.dropout_backward(dev(dy.astype(np.float32)), 0.2, 99, offset=13)).astype(np.float64)

    def loss(x):
        return float((dy * np.where(keep, x / 0.8, 0)).sum())
    slope = (loss(x + 1e-3 * v) - loss(x - 1e-3 * v)) / 2e-3
    # three roundings a term: dy, the scale and the product
    assert abs(slope - float((got * v).sum())) <= 4 * U * np.abs(got * v).sum() + 1e-9 * np.abs(dy).sum()


def test_dropout_offset_on_the_device(tcx):
    """A counter that a graph advances gives every replay its own mask."""
    from tensorcx_b200.graphs import CapturedSequence
    x = torch.ones(1003, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def body():
        y = tcx.dropout(x, 0.5, 21, offset=step)
        step.add_(x.numel())
        return y
    seq = CapturedSequence(body)
    step.zero_()
    for i in range(3):
        assert torch.equal(seq().clone(), tcx.dropout(x, 0.5, 21, offset=1003 * i)), i
    seq.release()


def test_dropout_on_another_stream(tcx):
    x = torch.randn(1 << 20, device="cuda")
    want = tcx.dropout(x, 0.1, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = x.clone()
        for _ in range(20):
            z = z * 1.0
        got = tcx.dropout(z, 0.1, 3)
    side.synchronize()
    assert torch.equal(got, want)


# ----------------------------------------------------------------------- layer norm
SHAPES = [(1, 1), (5, 1), (1, 2), (3, 5), (64, 31), (7, 127), (5, 128), (9, 260), (300, 64), (1000, 96), (4, 1001),
          (33, 1024), (6, 2048), (3, 2050), (2, 4096), (3, 4097), (150, 4096), (3, 6004), (5, 8192), (2, 8195),
          (2, 12000), (2, 16384), (3, 16385), (1, 32768), (2, 32770), (1, 40000), (2, 70001)]


def norm_case(rows, cols, residual, seed=0):
    rng = np.random.default_rng(rows * 1000003 + cols + seed)
    x = (rng.normal(size=(rows, cols)) * 3 + rng.normal(size=(rows, 1)) * 2).astype(np.float32)
    r = rng.normal(size=(rows, cols)).astype(np.float32) if residual else None
    w = rng.uniform(0.5, 1.5, cols).astype(np.float32)
    b = (rng.normal(size=cols) * 0.1).astype(np.float32)
    return x, r, w, b


def check_forward(y, mean, rstd, total, w, b, eps):
    t = total.astype(np.float64)
    n = t.shape[-1]
    k = n / 32 + 48  # additions in a row for a warp or more to a row, and the warp's and the block's trees
    m = t.mean(-1)
    var = t.var(-1)
    r = 1 / np.sqrt(var + np.float32(eps))
    spread = np.abs(t - m[..., None]).mean(-1)
    off_mean = k * U * spread + 2 * U * np.abs(m)
    # the deviations carry the roundings of the level that they are taken about
    rel_r = k * U / 2 + 8 * U + off_mean**2 * r * r + 2 * U * np.abs(m) * spread * r * r
    within(mean, m, off_mean, "mean")
    within(rstd, r, rel_r * r, "rstd")
    hat = (t - m[..., None]) * r[..., None]
    wd = np.ones(n) if w is None else np.abs(w.astype(np.float64))
    want = hat * (1 if w is None else w.astype(np.float64)) + (0 if b is None else b.astype(np.float64))
    bound = wd * (off_mean[..., None] * r[..., None] + np.abs(hat) * (rel_r[..., None] + 4 * U))
    bound = bound + 2 * U * np.abs(want) + 2 * U * (0 if b is None else np.abs(b.astype(np.float64)))
    within(y, want, bound, "y")


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("p,residual,affine", [(0.0, False, True), (0.1, True, True), (0.0, True, False),
                                               (0.25, False, True)])
def test_norm_forward(tcx, oracle, rows, cols, p, residual, affine):
    x, r, w, b = norm_case(rows, cols, residual)
    w, b = (w, b) if affine else (None, None)
    y, total, mean, rstd = tcx.layernorm_forward(
        dev(x), None if w is None else dev(w), None if b is None else dev(b),
        residual=None if r is None else dev(r), p=p, seed=17, offset=rows)
    want = x
    if p:
        want = np.where(keep_of(oracle, x.shape, p, 17, rows), x * scale_of(p), np.float32(0)).astype(np.float32)
    if residual:
        want = r + want
    assert host(total).tobytes() == want.tobytes()
    check_forward(host(y), host(mean), host(rstd), want, w, b, 1e-5)


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("cols", [36, 4096, 4097])
def test_norm_alignment(tcx, oracle, shift, cols):
    x, r, w, b = norm_case(5, cols, True)
    y, total, mean, rstd = tcx.layernorm_forward(dev(x, shift), dev(w, shift), dev(b), residual=dev(r, 4 - shift),
                                                 p=0.5, seed=1, offset=shift)
    want = r + np.where(keep_of(oracle, x.shape, 0.5, 1, shift), x * 2, np.float32(0)).astype(np.float32)
    assert host(total).tobytes() == want.tobytes()
    check_forward(host(y), host(mean), host(rstd), want, w, b, 1e-5)
    dy = np.random.default_rng(8).normal(size=x.shape).astype(np.float32)
    check_backward(tcx, oracle, dy, want, host(mean), host(rstd), w, r, 0.5, 1, shift, shift=shift)


def test_norm_leading_axes_and_empty(tcx):
    x = torch.randn(2, 3, 5, 40, device="cuda")
    y, total, mean, rstd = tcx.layernorm_forward(x)
    assert total is x and y.shape == x.shape and mean.shape == rstd.shape == (2, 3, 5)
    flat = tcx.layernorm_forward(x.view(30, 40))
    assert torch.equal(y.view(30, 40), flat[0]) and torch.equal(mean.view(30), flat[2])
    one = tcx.layernorm_forward(torch.randn(40, device="cuda"))
    assert one[2].shape == ()
    w = torch.ones(40, device="cuda")
    empty = torch.empty(0, 40, device="cuda")
    y, total, mean, rstd = tcx.layernorm_forward(empty, w, w)
    assert y.shape == (0, 40) and mean.shape == (0,)
    dx, dres, dw, db = tcx.layernorm_backward(empty, total, mean, rstd, w)
    assert dx.shape == (0, 40) and not dw.any() and not db.any()  # sums over no rows


@pytest.mark.parametrize("cols", [1, 7, 128, 4096, 4097, 16384, 40000])
def test_norm_constant_and_level_rows(tcx, cols):
    """Constant rows are exactly the bias; a level far above the spread costs no more than the
    level's own roundings."""
    x = np.stack([np.full(cols, v, np.float32) for v in (0.0, 0.3, -7.1, 1e30, 1e38)])
    b = np.linspace(-1, 1, cols).astype(np.float32)
    y, _, mean, rstd = tcx.layernorm_forward(dev(x), dev(np.full(cols, 1.5, np.float32)), dev(b))
    assert (host(y) == b).all()
    assert (host(mean) == x[:, 0]).all()
    assert np.allclose(host(rstd), 1 / math.sqrt(1e-5), rtol=1e-6)
    assert np.isnan(host(tcx.layernorm_forward(dev(x), eps=0.0)[0])).all()
    if cols > 1:
        t = (1e4 + np.random.default_rng(cols).normal(size=(4, cols))).astype(np.float32)
        y, _, mean, rstd = tcx.layernorm_forward(dev(t))
        check_forward(host(y), host(mean), host(rstd), t, None, None, 1e-5)


@pytest.mark.parametrize("cols", [5, 1024, 5000, 16384, 40000])
def test_norm_non_finite_rows_stay_their_own(tcx, cols):
    x = np.random.default_rng(cols).normal(size=(9, cols)).astype(np.float32)
    x[1, 0], x[4, cols // 2], x[7, cols - 1] = np.nan, np.inf, np.nan
    y, _, mean, rstd = tcx.layernorm_forward(dev(x))
    bad = np.zeros(9, bool)
    bad[[1, 4, 7]] = True
    y = host(y)
    assert np.isnan(y[bad]).all() and np.isfinite(y[~bad]).all()
    check_forward(y[~bad], host(mean)[~bad], host(rstd)[~bad], x[~bad], None, None, 1e-5)


def check_backward(tcx, oracle, dy, total, mean, rstd, w, dtotal, p, seed, offset, shift=0):
    rows, n = dy.shape
    dx, dres, dw, db = tcx.layernorm_backward(
        dev(dy, shift), dev(total, shift), dev(mean), dev(rstd), None if w is None else dev(w),
        dtotal=None if dtotal is None else dev(dtotal), p=p, seed=seed, offset=offset)
    d, t = dy.astype(np.float64), total.astype(np.float64)
    r = rstd.astype(np.float64)[:, None]
    hat = (t - mean.astype(np.float64)[:, None]) * r
    g = d if w is None else d * w.astype(np.float64)
    c1, c2 = g.mean(-1, keepdims=True), (g * hat).mean(-1, keepdims=True)
    want = r * (g - c1 - hat * c2)
    k = n / 32 + 48
    off1, off2 = k * U * np.abs(g).mean(-1, keepdims=True), (k + 4) * U * np.abs(g * hat).mean(-1, keepdims=True)
    bound = r * (off1 + np.abs(hat) * off2 + 6 * U * (np.abs(g) + np.abs(c1) + np.abs(hat * c2)))
    if dtotal is not None:
        want = want + dtotal.astype(np.float64)
    bound = bound + 2 * U * np.abs(want)
    within(host(dres), want, bound, "dresidual")
    if p:
        keep = keep_of(oracle, dy.shape, p, seed, offset)
        scale = float(scale_of(p))
        within(host(dx), np.where(keep, want * scale, 0),
               np.where(keep, bound * scale + 2 * U * np.abs(want) * scale, 0), "dx")
    else:
        assert dx is dres
    if w is None:
        assert dw is None and db is None
        return
    kr = rows + 8  # at worst all rows one after the other
    within(host(dw), (d * hat).sum(0), kr * U * np.abs(d * hat).sum(0), "dweight")
    within(host(db), d.sum(0), kr * U * np.abs(d).sum(0), "dbias")


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("p,dtotal,affine", [(0.0, False, True), (0.1, True, True), (0.0, True, False)])
def test_norm_backward(tcx, oracle, rows, cols, p, dtotal, affine):
    total, r, w, _ = norm_case(rows, cols, dtotal, seed=1)
    dy = np.random.default_rng(rows + cols).normal(size=(rows, cols)).astype(np.float32)
    t = total.astype(np.float64)
    mean = t.mean(-1).astype(np.float32)
    rstd = (1 / np.sqrt(t.var(-1) + 1e-5)).astype(np.float32)
    check_backward(tcx, oracle, dy, total, mean, rstd, w if affine else None, r, p, 23, cols)


@pytest.mark.parametrize("rows,cols", [(4096, 8), (5000, 33), (20000, 128), (3001, 300), (2000, 1000)])
def test_norm_backward_many_rows(tcx, oracle, rows, cols):
    """More rows than the grid holds at a time; the sums' order is fixed."""
    total, r, w, _ = norm_case(rows, cols, True, seed=2)
    dy = np.random.default_rng(rows).normal(size=(rows, cols)).astype(np.float32)
    t = total.astype(np.float64)
    mean, rstd = t.mean(-1).astype(np.float32), (1 / np.sqrt(t.var(-1) + 1e-5)).astype(np.float32)
    check_backward(tcx, oracle, dy, total, mean, rstd, w, r, 0.1, 5, 0)
    args = [dev(v) for v in (dy, total, mean, rstd, w)]
    first = [host(v) for v in tcx.layernorm_backward(*args)]
    again = [host(v) for v in tcx.layernorm_backward(*args)]
    assert all(a.tobytes() == b.tobytes() for a, b in zip(first, again))


@pytest.mark.parametrize("rows,cols", [(310, 16500), (160, 20001), (200, 16384), (90, 33001)])
def test_norm_long_rows_in_turn(tcx, oracle, rows, cols):
    """More long rows than run at a time: a block, or a cluster of them, takes several."""
    x, r, w, b = norm_case(rows, cols, True, seed=3)
    y, total, mean, rstd = tcx.layernorm_forward(dev(x), dev(w), dev(b))
    check_forward(host(y), host(mean), host(rstd), x, w, b, 1e-5)
    y, total, mean, rstd = tcx.layernorm_forward(dev(x), dev(w), dev(b), residual=dev(r), p=0.5, seed=9, offset=1)
    want = r + np.where(keep_of(oracle, x.shape, 0.5, 9, 1), x * 2, np.float32(0)).astype(np.float32)
    assert host(total).tobytes() == want.tobytes()
    check_forward(host(y), host(mean), host(rstd), want, w, b, 1e-5)
    dy = np.random.default_rng(rows).normal(size=x.shape).astype(np.float32)
    check_backward(tcx, oracle, dy, want, host(mean), host(rstd), w, x, 0.5, 9, 1)


@pytest.mark.parametrize("rows,cols", [(310, 8192), (350, 6001), (1790, 6404), (1801, 1101), (1777, 8403),
                                       (1800, 10000), (1790, 17408)])
def test_norm_many_middling_rows(tcx, oracle, rows, cols):
    """Rows of one block, enough of them that fewer warps take more words of each."""
    test_norm_long_rows_in_turn(tcx, oracle, rows, cols)


@pytest.mark.parametrize("rows,cols", [(60001, 1), (60000, 2), (60002, 31), (31001, 64), (40003, 67), (20001, 128),
                                       (20003, 129), (10001, 256), (10003, 259)])
def test_norm_many_short_rows(tcx, oracle, rows, cols):
    """Rows that share a warp, more of them than run at a time, and the last warp not full."""
    test_norm_long_rows_in_turn(tcx, oracle, rows, cols)


@pytest.mark.parametrize("cols", [3, 130])
def test_norm_gradient_against_differences(tcx, oracle, cols):
    """The kernels' gradients along a direction against central differences of the 64-bit
    formula: loss = sum(dy y) + sum(dtotal total)."""
    rows, p, eps = 6, 0.3, 1e-5
    rng = np.random.default_rng(cols)
    x, r, dy, dt = (rng.normal(size=(rows, cols)) for _ in range(4))
    w, b = rng.uniform(0.5, 1.5, cols), rng.normal(size=cols)
    keep = keep_of(oracle, x.shape, p, 3, 0)
    y, total, mean, rstd = tcx.layernorm_forward(*(dev(v.astype(np.float32)) for v in (x, w, b)), eps,
                                                 residual=dev(r.astype(np.float32)), p=p, seed=3)
    grads = tcx.layernorm_backward(dev(dy.astype(np.float32)), total, mean, rstd, dev(w.astype(np.float32)),
                                   dtotal=dev(dt.astype(np.float32)), p=p, seed=3)

    def loss(x, r, w, b):
        t = r + np.where(keep, x / (1 - p), 0)
        hat = (t - t.mean(-1, keepdims=True)) / np.sqrt(t.var(-1, keepdims=True) + eps)
        return float((dy * (hat * w + b)).sum() + (dt * t).sum())
    point = [x, r, w, b]
    for i, g in enumerate(grads):
        v = rng.normal(size=point[i].shape)
        h = 1e-5
        up, down = (loss(*[q + s * h * v if j == i else q for j, q in enumerate(point)]) for s in (1, -1))
        g = host(g).astype(np.float64)
        # a float32 gradient of a float32 point: some tens of roundings of each term; a difference's own error is h^2
        size = np.abs(g * v).sum() + np.abs(dy).sum()
        assert abs((up - down) / (2 * h) - float((g * v).sum())) <= 200 * U * size + 1e-7 * size, i


# ----------------------------------------------------------------------- recurrence
RSHAPES = [(1, 1, 1), (3, 1, 5), (5, 1, 1001), (300, 1, 64), (2, 2, 3), (2, 5, 3), (1, 7, 128), (4, 17, 260),
           (1, 64, 128), (3, 65, 130), (2, 257, 33), (1, 300, 1024), (1, 1000, 256), (2, 1025, 68), (1, 5000, 4), (9, 129, 512), (1, 2049, 127),
           (70, 33, 1000)]


def recurrence_case(batch, time, channels, form, seed=0):
    rng = np.random.default_rng(batch * 7919 + time * 104729 + channels + seed)
    shape = (batch, time, channels)
    gate = rng.uniform(-1, 1, shape) if form == "decay" else rng.normal(size=shape) * 2 + 1
    x, dh = rng.normal(size=shape), rng.normal(size=shape)
    init, dstate = rng.normal(size=(batch, channels)), rng.normal(size=(batch, channels))
    return tuple(v.astype(np.float32) for v in (gate, x, init, dh, dstate))


def gates(gate, form):
    g = gate.astype(np.float64)
    if form == "decay":
        return g, np.ones_like(g)
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-g)), 1 / (1 + np.exp(g))


def roundings(gate, form):
    """Roundings that one step adds to a term on its way: a product and a sum, and in the
    sigmoid form those of the gate (an exponential whose argument was rounded, a sum, a
    quotient, a product)."""
    live = np.abs(gate[np.isfinite(gate)])
    return 4.0 if form == "decay" else 24.0 + 2 * (live.max() if live.size else 0)


def scan(a, b, start, live, kappa):
    """h, and a bound of any evaluation of it that multiplies and adds along the steps: each
    term is rounded at most kappa times for each step that it has gone through."""
    h, m = start.astype(np.float64), np.abs(start.astype(np.float64))
    e = np.zeros_like(m)
    hs, es = np.empty(a.shape), np.empty(a.shape)
    for t in range(a.shape[1]):
        on = live[:, t, None]
        at, bt = np.where(on, a[:, t], 1.0), np.where(on, b[:, t], 0.0)
        e = np.abs(at) * (e + kappa * U * m)
        m = np.abs(at) * m + np.abs(bt)
        h = at * h + bt
        hs[:, t], es[:, t] = h, e + 2 * kappa * U * m
    return hs, es


def live_steps(batch, time, lengths):
    n = np.full(batch, time) if lengths is None else np.clip(lengths, 0, time)
    return np.arange(time)[None, :] < n[:, None]


def check_recurrence(tcx, gate, x, init, dh, dstate, form, lengths=None, shift=0):
    batch, time, channels = gate.shape
    a, rest = gates(gate, form)
    kappa = roundings(gate, form)
    live = live_steps(batch, time, lengths)
    n = None if lengths is None else dev(lengths.astype(np.int32))
    h, state = tcx.gated_recurrence(dev(gate, shift), dev(x, shift), None if init is None else dev(init, shift),
                                    form=form, lengths=n)
    start = np.zeros((batch, channels)) if init is None else init.astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, bound = scan(a, rest * x.astype(np.float64), start, live, kappa)
    within(host(h), want, bound, "h")
    if time:
        within(host(state), want[:, -1], bound[:, -1], "state")
    else:
        assert (host(state) == start).all()
    # backward from float32 values of h
    hs = want.astype(np.float32)
    got = tcx.gated_recurrence_backward(
        dev(dh, shift), dev(gate, shift), dev(x, shift) if form == "sigmoid" else None, dev(hs, shift),
        None if init is None else dev(init, shift), form=form, lengths=n,
        dstate=None if dstate is None else dev(dstate, shift))
    end = np.zeros((batch, channels)) if dstate is None else dstate.astype(np.float64)
    d = dh.astype(np.float64)
    on = live[:, :, None]
    with np.errstate(invalid="ignore"):
        aa = np.where(on, a, 1.0)
        flip = slice(None, None, -1)
        c, off = scan(aa[:, flip], (aa * d)[:, flip], end, np.ones_like(live), kappa)
    c, off = c[:, flip], off[:, flip]
    after = np.concatenate([c[:, 1:], end[:, None]], 1) if time else c
    off_after = np.concatenate([off[:, 1:], np.zeros((batch, 1, channels))], 1) if time else off
    g = d + after
    off_g = off_after + 2 * U * (np.abs(d) + np.abs(after))
    before = np.concatenate([start[:, None], hs[:, :-1].astype(np.float64)], 1) if time else hs
    with np.errstate(invalid="ignore"):
        factor = before if form == "decay" else (before - x.astype(np.float64)) * a * rest
        dgate, dx = np.where(on, g * factor, 0), np.where(on, g * rest, 0)
        bg = np.where(on, off_g * np.abs(factor) + 2 * kappa * U * np.abs(g * factor), 0)
        bx = np.where(on, off_g * rest + 2 * kappa * U * np.abs(g * rest), 0)
    within(host(got[0]), dgate, bg, "dgate")
    within(host(got[1]), dx, bx, "dx")
    if init is None:
        assert got[2] is None
    else:
        within(host(got[2]), c[:, 0] if time else end, off[:, 0] + U * np.abs(c[:, 0]) if time else 0 * end, "dinitial")


@pytest.mark.parametrize("batch,time,channels", RSHAPES)
@pytest.mark.parametrize("form", ["decay", "sigmoid"])
@pytest.mark.parametrize("carried", [True, False])
def test_recurrence(tcx, batch, time, channels, form, carried):
    gate, x, init, dh, dstate = recurrence_case(batch, time, channels, form)
    check_recurrence(tcx, gate, x, init if carried else None, dh, dstate if carried else None, form)


@pytest.mark.parametrize("form", ["decay", "sigmoid"])
@pytest.mark.parametrize("time,channels", [(1, 7), (37, 40), (700, 132), (1500, 257)])
def test_recurrence_lengths(tcx, form, time, channels):
    """Padded steps hold the state and take no gradient, whatever stands there; lengths are
    clamped to the batch's."""
    batch = 6
    gate, x, init, dh, dstate = recurrence_case(batch, time, channels, form, seed=1)
    lengths = np.array([0, 1, time // 2, time, time + 5, -3])
    pad = ~live_steps(batch, time, lengths)
    gate[pad], x[pad] = np.nan, np.inf
    check_recurrence(tcx, gate, x, init, dh, dstate, form, lengths)
    h, state = tcx.gated_recurrence(dev(gate), dev(x), dev(init), form=form, lengths=dev(lengths.astype(np.int32)))
    h = host(h)
    for b, n in enumerate(np.clip(lengths, 0, time)):
        held = h[b, n - 1] if n else init[b]
        assert (h[b, n:] == held).all() and (host(state)[b] == (h[b, -1])).all()


@pytest.mark.parametrize("form", ["decay", "sigmoid"])
@pytest.mark.parametrize("batch,time,channels", [(300, 300, 20), (250, 140, 21), (300, 40, 600), (700, 100, 301)])
def test_recurrence_many_sequences(tcx, form, batch, time, channels):
    """Enough sequences to fill the machine, of different lengths: whole ones to a block, or a
    thread to a channel."""
    gate, x, init, dh, dstate = recurrence_case(batch, time, channels, form, seed=6)
    lengths = np.random.default_rng(batch).integers(-1, time + 2, batch)
    pad = ~live_steps(batch, time, lengths)
    gate[pad], x[pad] = np.nan, np.inf
    check_recurrence(tcx, gate, x, init, dh, dstate, form, lengths)
    h, _ = tcx.gated_recurrence(dev(gate), dev(x), dev(init), form=form, lengths=dev(lengths.astype(np.int32)))
    h = host(h)
    for b, n in enumerate(np.clip(lengths, 0, time)):
        assert (h[b, n:] == (h[b, n - 1] if n else init[b])).all()


@pytest.mark.parametrize("form", ["decay", "sigmoid"])
@pytest.mark.parametrize("lengths", [False, True])
@pytest.mark.parametrize("batch,channels,shift", [(1, 3, 0), (4, 1001, 0), (37, 33, 0), (300, 256, 0), (12, 1001, 1)])
def test_recurrence_one_step(tcx, form, lengths, batch, channels, shift):
    """The batch's channels as one row, or each entry's by its length."""
    gate, x, init, dh, dstate = recurrence_case(batch, 1, channels, form, seed=8)
    n = np.random.default_rng(batch).integers(-1, 3, batch) if lengths else None
    if lengths:
        pad = ~live_steps(batch, 1, n)
        gate[pad], x[pad] = np.nan, np.inf
    check_recurrence(tcx, gate, x, init, dh, dstate, form, n, shift=shift)


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("channels", [128, 96, 33])
def test_recurrence_alignment(tcx, shift, channels):
    gate, x, init, dh, dstate = recurrence_case(2, 150, channels, "sigmoid", seed=2)
    check_recurrence(tcx, gate, x, init, dh, dstate, "sigmoid", shift=shift)


@pytest.mark.parametrize("shape", [(0, 5, 4), (2, 0, 4), (2, 5, 0), (0, 0, 0)])
@pytest.mark.parametrize("form", ["decay", "sigmoid"])
def test_recurrence_empty(tcx, shape, form):
    gate, x, init, dh, dstate = recurrence_case(*shape, form)
    h, state = tcx.gated_recurrence(dev(gate), dev(x), dev(init), form=form)
    assert tuple(h.shape) == shape and (host(state) == init).all()
    dgate, dx, dinit = tcx.gated_recurrence_backward(dev(dh), dev(gate), dev(x), h, dev(init), form=form,
                                                     dstate=dev(dstate))
    assert tuple(dx.shape) == shape and (host(dinit) == dstate).all()


def test_recurrence_gates_at_the_ends(tcx):
    """Gates of 0 forget everything, gates of 1 keep everything, logits far out saturate
    without NaN, and a forgotten NaN of another channel stays there."""
    time, ch = 500, 36
    x = np.random.default_rng(0).normal(size=(1, time, ch)).astype(np.float32)
    zeros, ones = np.zeros_like(x), np.ones_like(x)
    init = np.ones((1, ch), np.float32)
    assert (host(tcx.gated_recurrence(dev(zeros), dev(x), dev(init))[0]) == x).all()
    assert (host(tcx.gated_recurrence(dev(ones), dev(zeros), dev(init))[0]) == 1).all()
    for z, want in ((200.0, 1.0), (-200.0, None), (np.inf, 1.0), (-np.inf, None)):
        h = host(tcx.gated_recurrence(dev(np.full_like(x, z)), dev(x), dev(init), form="sigmoid")[0])
        assert (h == (x if want is None else want)).all(), z
    x[0, 100, 3] = np.nan
    h = host(tcx.gated_recurrence(dev(ones * 0.5), dev(x), dev(init))[0])
    assert np.isnan(h[0, 100:, 3]).all() and np.isnan(h).sum() == time - 100
    # gates above one from a zero state: the products overflow, the state stays zero
    big = host(tcx.gated_recurrence(dev(ones * 3), dev(zeros))[0])
    assert not big.any()


@pytest.mark.parametrize("form", ["decay", "sigmoid"])
def test_recurrence_gradient_against_differences(tcx, form):
    gate, x, init, dh, dstate = recurrence_case(2, 90, 5, form, seed=3)
    lengths = np.array([90, 41])
    live = live_steps(2, 90, lengths)
    n = dev(lengths.astype(np.int32))
    h, state = tcx.gated_recurrence(dev(gate), dev(x), dev(init), form=form, lengths=n)
    grads = tcx.gated_recurrence_backward(dev(dh), dev(gate), dev(x), h, dev(init), form=form, lengths=n,
                                          dstate=dev(dstate))

    def loss(gate, x, init):
        a, rest = (gate, 1.0) if form == "decay" else (1 / (1 + np.exp(-gate)), 1 / (1 + np.exp(gate)))
        hs, _ = scan(a, rest * x, init, live, 0)
        return float((dh * hs).sum() + (dstate * hs[:, -1]).sum())
    point = [v.astype(np.float64) for v in (gate, x, init)]
    rng = np.random.default_rng(9)
    for i, g in enumerate(grads):
        v = rng.normal(size=point[i].shape)
        step = 1e-5
        up, down = (loss(*[q + s * step * v if j == i else q for j, q in enumerate(point)]) for s in (1, -1))
        g = host(g).astype(np.float64)
        size = np.abs(g * v).sum() + np.abs(dh).sum()
        assert abs((up - down) / (2 * step) - float((g * v).sum())) <= 200 * U * size + 1e-7 * size, i


@pytest.mark.parametrize("form", ["decay", "sigmoid"])
def test_recurrence_in_parts_is_the_whole(tcx, form):
    """A sequence in two calls, then token by token, goes on from the state."""
    gate, x, init, _, _ = recurrence_case(3, 400, 72, form, seed=4)
    kappa = roundings(gate, form)
    a, rest = gates(gate, form)
    want, bound = scan(a, rest * x, init, live_steps(3, 400, None), kappa)
    g, xs = dev(gate), dev(x)
    h1, state = tcx.gated_recurrence(g[:, :390].contiguous(), xs[:, :390].contiguous(), dev(init), form=form)
    parts = [h1]
    for t in range(390, 400):
        h, state = tcx.gated_recurrence(g[:, t:t + 1].contiguous(), xs[:, t:t + 1].contiguous(), state, form=form)
        parts.append(h)
    within(host(torch.cat(parts, 1)), want, bound, "parts")
    assert torch.equal(state, parts[-1][:, 0])


def test_recurrence_same_bits_every_time(tcx):
    gate, x, init, dh, dstate = (dev(v) for v in recurrence_case(1, 20000, 192, "sigmoid", seed=5))
    first = tcx.gated_recurrence(gate, x, init, form="sigmoid")
    back = tcx.gated_recurrence_backward(dh, gate, x, first[0], init, form="sigmoid", dstate=dstate)
    for _ in range(10):
        again = tcx.gated_recurrence(gate, x, init, form="sigmoid")
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        grads = tcx.gated_recurrence_backward(dh, gate, x, first[0], init, form="sigmoid", dstate=dstate)
        assert all(torch.equal(a, b) for a, b in zip(back, grads))


# ------------------------------------------------------------------------ large sizes
def test_places_past_32_bits(tcx):
    """Tensors of more than 2^31 elements: the last rows and steps against the same rows alone."""
    rows, cols = (1 << 19) + 3, 4100
    x = torch.randn(rows, cols, device="cuda")
    last = x[-2:].contiguous()
    at = (rows - 2) * cols
    y = tcx.dropout(x, 0.5, 77)
    assert torch.equal(y[-2:], tcx.dropout(last, 0.5, 77, offset=at))
    del y
    torch.cuda.empty_cache()
    w = torch.rand(cols, device="cuda")
    y, total, mean, rstd = tcx.layernorm_forward(x, w, w, p=0.5, seed=77)
    small = tcx.layernorm_forward(last, w, w, p=0.5, seed=77, offset=at)
    for a, b in zip((y, total, mean, rstd), small):
        assert torch.equal(a[-2:], b)
    dx, dres, _, _ = tcx.layernorm_backward(x, total, mean, rstd, w, p=0.5, seed=77)
    sdx, sres, _, _ = tcx.layernorm_backward(last, small[1], small[2], small[3], w, p=0.5, seed=77, offset=at)
    assert torch.equal(dx[-2:], sdx) and torch.equal(dres[-2:], sres)
    del x, y, total, mean, rstd, dx, dres
    torch.cuda.empty_cache()
    batch, time, ch = 3, 70001, 10240
    gate, x = torch.rand(batch, time, ch, device="cuda"), torch.randn(batch, time, ch, device="cuda")
    h, state = tcx.gated_recurrence(gate, x)
    tail = 3000  # gates below one: what came before is forgotten
    part = tcx.gated_recurrence(gate[-1:, -tail:].contiguous(), x[-1:, -tail:].contiguous(),
                                h[-1:, -tail - 1].contiguous())
    assert torch.allclose(h[-1:, -tail:], part[0], rtol=1e-4, atol=1e-4)
    assert torch.allclose(state[-1:], part[1], rtol=1e-4, atol=1e-4)
    dgate, dx, _ = tcx.gated_recurrence_backward(x, gate, None, h)
    want = tcx.gated_recurrence_backward(x[-1:, -tail:].contiguous(), gate[-1:, -tail:].contiguous(), None,
                                         part[0], h[-1:, -tail - 1].contiguous())
    assert torch.allclose(dgate[-1:, -tail:], want[0], rtol=1e-3, atol=1e-3)
    assert torch.allclose(dx[-1:, -tail:], want[1], rtol=1e-4, atol=1e-4)
    del gate, x, h, state, part, dgate, dx, want
    torch.cuda.empty_cache()


# --------------------------------------------------------------------------- refusals
def test_refusals(tcx):
    x = torch.randn(4, 6, device="cuda")
    w = torch.ones(6, device="cuda")
    stat = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError, match="probability"):
        tcx.dropout(x, 1.5, 0)
    with pytest.raises(ValueError, match="probability"):
        tcx.dropout(x, float("nan"), 0)
    with pytest.raises(TypeError, match="probability"):
        tcx.dropout(x, True, 0)
    with pytest.raises(ValueError, match="seed"):
        tcx.dropout(x, 0.5, None)
    with pytest.raises(ValueError, match="seed"):
        tcx.dropout(x, 0.5, -1)
    with pytest.raises(ValueError, match="offset"):
        tcx.dropout(x, 0.5, 1, offset=-1)
    with pytest.raises(ValueError, match="offset"):
        tcx.dropout(x, 0.5, 1, offset=torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="offset"):
        tcx.dropout(x, 0.5, 1, offset=torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="shape"):
        tcx.dropout(x, 0.5, 1, residual=w)
    with pytest.raises(ValueError, match="contiguous"):
        tcx.dropout(x.t(), 0.5, 1)
    with pytest.raises(ValueError, match="float32"):
        tcx.dropout(x.double(), 0.5, 1)
    with pytest.raises(ValueError, match="device"):
        tcx.dropout(x.cpu(), 0.5, 1)
    with pytest.raises(TypeError):
        tcx.dropout([1.0], 0.5, 1)
    with pytest.raises(ValueError, match="shape"):
        tcx.layernorm_forward(x, stat)
    with pytest.raises(ValueError, match="epsilon"):
        tcx.layernorm_forward(x, eps=-1.0)
    with pytest.raises(ValueError, match="seed"):
        tcx.layernorm_forward(x, p=0.1)
    with pytest.raises(ValueError, match="last axis"):
        tcx.layernorm_forward(torch.empty(3, 0, device="cuda"))
    with pytest.raises(ValueError, match="last axis"):
        tcx.layernorm_forward(torch.tensor(1.0, device="cuda"))
    with pytest.raises(ValueError, match="shape"):
        tcx.layernorm_backward(x, x, w, stat, w)
    with pytest.raises(ValueError, match="shape"):
        tcx.layernorm_backward(x[:3], x, stat, stat, w)
    g = torch.rand(2, 3, 4, device="cuda")
    with pytest.raises(ValueError, match="form"):
        tcx.gated_recurrence(g, g, form="tanh")
    with pytest.raises(ValueError, match="time"):
        tcx.gated_recurrence(x, x)
    with pytest.raises(ValueError, match="shape"):
        tcx.gated_recurrence(g, g[:, :2].contiguous())
    with pytest.raises(ValueError, match="shape"):
        tcx.gated_recurrence(g, g, x)
    with pytest.raises(ValueError, match="lengths"):
        tcx.gated_recurrence(g, g, lengths=torch.ones(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="lengths"):
        tcx.gated_recurrence(g, g, lengths=torch.ones(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        tcx.gated_recurrence(g, None)
    with pytest.raises(ValueError, match="needs x"):
        tcx.gated_recurrence_backward(g, g, None, g, form="sigmoid")
    with pytest.raises(ValueError, match="shape"):
        tcx.gated_recurrence_backward(g, g, None, g, dstate=x)
