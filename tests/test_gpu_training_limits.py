"""The training operators where their arguments end: places of the random stream at 2^64, outputs
that a call without dropout need not have, sums over many rows, rows of the widest spread, the largest gates,
buffers at any address, host threads and streams.

The masks are compared with the generator's definition in whole-number arithmetic on the host.
"""
import threading

import numpy as np
import pytest
import torch

from test_gpu_training import (check_backward, check_forward, check_recurrence, dev, host, keep_of,
                               live_steps, norm_case, recurrence_case, roundings, scale_of, scan, within)

pytestmark = pytest.mark.gpu

U = 2.0**-24


def mask_at(shape, p, seed, offset):
    """keep of every element, its place taken modulo 2^64 (Philox4x32-10, word place % 4 of the
    block place / 4)."""
    place = np.arange(int(np.prod(shape)), dtype=np.uint64) + np.uint64(offset % 2**64)
    block, half, low = place >> np.uint64(2), np.uint64(32), np.uint64(0xFFFFFFFF)
    c = [block & low, block >> half, np.zeros_like(block), np.zeros_like(block)]
    k0, k1 = seed % 2**32, seed >> 32
    for r in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64((k0 + r * 0x9E3779B9) % 2**32), b & low,
             (a >> half) ^ c[3] ^ np.uint64((k1 + r * 0xBB67AE85) % 2**32), a & low]
    word = np.choose((place & np.uint64(3)).astype(np.int64), c) >> np.uint64(8)
    return (word.astype(np.float64) * 2.0**-24 >= p).reshape(shape)


# ------------------------------------------------------------- the end of the stream
@pytest.mark.parametrize("rows,cols", [(2, 256), (5, 255), (40, 33), (3, 64), (7, 8192), (4, 4099)])
@pytest.mark.parametrize("before", [1, 2, 64, 67, 515])
def test_one_mask_past_the_stream_s_end(tcx, rows, cols, before):
    """Place 2^64 is place 0 in every kernel: dropout, the norm and its gradient, aligned buffers
    or not, the offset given on the host or by a counter of -`before` on the device."""
    p, seed, offset = 0.5, 91, 2**64 - before
    x, r, w, b = norm_case(rows, cols, True)
    keep = mask_at(x.shape, p, seed, offset)
    want = np.where(keep, x * scale_of(p), np.float32(0)).astype(np.float32)
    total = r + want
    counter = torch.tensor([-before], dtype=torch.int64, device="cuda")
    dy = np.random.default_rng(before).normal(size=x.shape).astype(np.float32)
    for at in (offset, counter):
        for shift in (0, 1):
            assert host(tcx.dropout(dev(x, shift), p, seed, offset=at)).tobytes() == want.tobytes()
            y, got, mean, rstd = tcx.layernorm_forward(dev(x, shift), dev(w), dev(b), residual=dev(r, shift), p=p,
                                                       seed=seed, offset=at)
            assert host(got).tobytes() == total.tobytes()
            dx, dres, _, _ = tcx.layernorm_backward(dev(dy, shift), got, mean, rstd, dev(w), p=p, seed=seed, offset=at)
            dx, dres = host(dx), host(dres)
            assert dx.tobytes() == np.where(keep, dres * scale_of(p), np.float32(0)).astype(np.float32).tobytes()


# ------------------------------------------------------- outputs that are other tensors' copies
@pytest.mark.parametrize("rows,cols", [(1, 1), (37, 100), (300, 4097), (2, 40000)])
@pytest.mark.parametrize("shift", [0, 3])
def test_outputs_given_are_written(tcx, rows, cols, shift):
    """Without dropout and residual the total is the input, and the input's gradient is the
    residual's: a C caller may pass NULL for them, and finds them in a buffer that it passes."""
    from tensorcx_b200 import _abi
    x, _, w, b = norm_case(rows, cols, False)
    xd, wd, bd = dev(x, shift), dev(w), dev(b)
    y, mean, rstd = torch.empty_like(xd), *(torch.empty(rows, device="cuda") for _ in range(2))
    total, dx, dres = (torch.full_like(xd, float("nan")) for _ in range(3))
    stream = torch.cuda.current_stream().cuda_stream
    assert _abi.lib().tcx_sm100_layernorm_forward(
        stream, xd.data_ptr(), None, wd.data_ptr(), bd.data_ptr(), y.data_ptr(), total.data_ptr(), mean.data_ptr(),
        rstd.data_ptr(), rows, cols, 1e-5, 0.0, 0, 0, None) == _abi.OK
    want = tcx.layernorm_forward(xd, wd, bd)
    assert host(total).tobytes() == x.tobytes()
    assert all(torch.equal(a, c) for a, c in zip((y, mean, rstd), (want[0], want[2], want[3])))
    assert _abi.lib().tcx_sm100_layernorm_backward(
        stream, y.data_ptr(), total.data_ptr(), mean.data_ptr(), rstd.data_ptr(), wd.data_ptr(), None, dres.data_ptr(),
        dx.data_ptr(), None, None, rows, cols, 0.0, 0, 0, None, None, 0) == _abi.OK
    assert torch.equal(dx, dres) and torch.isfinite(dx).all()
    # the input itself as the total's buffer, and the residual's gradient as the input's
    assert _abi.lib().tcx_sm100_layernorm_forward(
        stream, xd.data_ptr(), None, wd.data_ptr(), bd.data_ptr(), y.data_ptr(), xd.data_ptr(), mean.data_ptr(),
        rstd.data_ptr(), rows, cols, 1e-5, 0.0, 0, 0, None) == _abi.OK
    assert host(xd).tobytes() == x.tobytes() and torch.equal(y, want[0])


# ------------------------------------------------------------------ sums over many rows
def chain(rows, held):
    """Roundings that a term of a column's sum goes through where the sums are a pass of their own:
    three of its own, the rows of a span of 16 one after the other, the spans' sums of one of the
    `held` parts of the rows, and the parts' sums (at most 592, by 32 warps, then theirs)."""
    return 3 + 16 + -(-rows // (16 * held)) + 19 + 10


def chain_in_registers(rows, held):
    """The same where they are added on the way: three of its own, a group of warps' 128 rows (144
    where the blocks are a multiple of four), the sums of up to 32 groups, and the blocks' (20 of
    a warp's every 32nd, the twenties, and the warps')."""
    blocks = max(600, rows // 128 + 600)
    return 3 + min(144, -(-rows // held)) + 10 + 20 + -(-blocks // 640) + 10


def column_sums(tcx, dy, total, mean, rstd, rows, k):
    """dweight and dbias against 64 bits; all on the GPU."""
    w = torch.ones(dy.shape[1], device="cuda")
    _, _, dw, db = tcx.layernorm_backward(dy, total, mean, rstd, w)
    exact_w, size_w = (torch.zeros(dy.shape[1], dtype=torch.float64, device="cuda") for _ in range(2))
    exact_b, size_b = torch.zeros_like(exact_w), torch.zeros_like(exact_w)
    for i in range(0, rows, 1 << 14):
        d = dy[i:i + (1 << 14)].double()
        term = d * (total[i:i + (1 << 14)].double() - mean[i:i + (1 << 14), None]) * rstd[i:i + (1 << 14), None]
        exact_w += term.sum(0)
        size_w += term.abs().sum(0)
        exact_b += d.sum(0)
        size_b += d.abs().sum(0)
    within(host(dw), host(exact_w), k * U * host(size_w), "dweight")
    within(host(db), host(exact_b), k * U * host(size_b), "dbias")


def many_rows(rows, cols, shift, value):
    """A constant gradient (its roundings all go one way as a sum grows) and random rows."""
    def at_shift(t):
        buf = torch.empty(t.numel() + shift, device="cuda")
        buf[shift:] = t.reshape(-1)
        return buf[shift:].view(t.shape)
    make = torch.Generator(device="cuda").manual_seed(rows + cols)
    total = at_shift(torch.randn(rows, cols, generator=make, device="cuda"))
    rstd = 1 / total.std(1, correction=0)
    return at_shift(torch.full((rows, cols), value, device="cuda")), total, total.mean(1), rstd


@pytest.mark.parametrize("rows,cols,value", [(1000000, 64, 0.1), (700003, 129, 0.7), (1100, 40, 0.1),
                                             (30000, 4099, 0.3)])
def test_column_sums_of_many_rows_at_any_address(tcx, rows, cols, value):
    column_sums(tcx, *many_rows(rows, cols, 1, value), rows, chain(rows, 592 if cols < 256 else 64))


@pytest.mark.parametrize("rows,cols", [(3001, 67), (1300, 4097), (1100, 40), (2400, 12)])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_many_rows_at_any_address(tcx, oracle, rows, cols, shift):
    """Blocks take several rows in turn, and splits of the rows may be empty."""
    x, r, w, b = norm_case(rows, cols, True, seed=5)
    y, total, mean, rstd = tcx.layernorm_forward(dev(x, shift), dev(w), dev(b))
    check_forward(host(y), host(mean), host(rstd), x, w, b, 1e-5)
    y, total, mean, rstd = tcx.layernorm_forward(dev(x, shift), dev(w, shift), dev(b), residual=dev(r, shift), p=0.5,
                                                 seed=2, offset=shift)
    want = r + np.where(keep_of(oracle, x.shape, 0.5, 2, shift), x * 2, np.float32(0)).astype(np.float32)
    assert host(total).tobytes() == want.tobytes()
    check_forward(host(y), host(mean), host(rstd), want, w, b, 1e-5)
    dy = np.random.default_rng(rows).normal(size=x.shape).astype(np.float32)
    check_backward(tcx, oracle, dy, want, host(mean), host(rstd), w, x, 0.5, 2, shift, shift=shift)


@pytest.mark.parametrize("rows,cols,held,value", [
    (18000000, 8, 14208, 0.8738095), (6000000, 100, 4736, 0.8738095), (3000001, 509, 2368, 0.8738095),
    (1500000, 1024, 1184, 0.8738095), (750000, 2050, 592, 0.8738095), (190001, 4100, 148, 0.8738095),
    (190000, 8192, 148, 0.8738095), (70000, 16388, 32, 0.8738095), (2369, 512, 2368, 0.1), (20000, 4097, 148, 0.7)])
def test_column_sums_of_many_rows(tcx, rows, cols, held, value):
    """More than a thousand rows to each place that the GPU has for them, and a few."""
    column_sums(tcx, *many_rows(rows, cols, 0, value), rows, chain_in_registers(rows, held))
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,cols", [(160004, 1001), (20004, 8190), (5000, 16385)])
def test_rounds_of_blocks_are_one_call(tcx, rows, cols):
    """More rows than one round of blocks takes, with dropout and dtotal: the last rows (from a
    multiple of 4 on) are those of a call on them alone, the sums the parts' sums."""
    make = torch.Generator(device="cuda").manual_seed(cols)
    dy, total, extra = (torch.randn(rows, cols, generator=make, device="cuda") for _ in range(3))
    mean, rstd, w = total.mean(1), 1 / total.std(1, correction=0), torch.ones(cols, device="cuda")
    kw = dict(p=0.25, seed=6)
    dx, dres, dw, db = tcx.layernorm_backward(dy, total, mean, rstd, w, dtotal=extra, offset=9, **kw)
    cut = rows // 2 // 4 * 4
    parts = [tcx.layernorm_backward(dy[s], total[s], mean[s].contiguous(), rstd[s].contiguous(), w, dtotal=extra[s],
                                    offset=9 + s.start * cols, **kw) for s in (slice(0, cut), slice(cut, rows))]
    assert torch.equal(dx, torch.cat([q[0] for q in parts])) and torch.equal(dres, torch.cat([q[1] for q in parts]))
    k = 2 * chain_in_registers(rows, 32)
    size_w, size_b = (dy * (total - mean[:, None]) * rstd[:, None]).abs().sum(0), dy.abs().sum(0)
    within(host(dw), host(parts[0][2].double() + parts[1][2].double()), k * U * host(size_w), "dweight")
    within(host(db), host(parts[0][3].double() + parts[1][3].double()), k * U * host(size_b), "dbias")
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------- wide rows
@pytest.mark.parametrize("cols", [2, 40, 1024, 5000, 16384, 40000])
@pytest.mark.parametrize("shift", [0, 1])
def test_norm_of_rows_of_the_widest_spread(tcx, cols, shift):
    """Deviations whose squares sum to half of what a float32 holds, about levels near and far,
    next to an ordinary row."""
    t = np.random.default_rng(cols).normal(size=(4, cols))
    t -= t.mean(1, keepdims=True)
    t *= np.sqrt(1.7e38) / np.sqrt((t * t).sum(1, keepdims=True))
    t[1] += 1e19
    t[2] *= 1e-19
    t = t.astype(np.float32)
    y, _, mean, rstd = tcx.layernorm_forward(dev(t, shift))
    check_forward(host(y), host(mean), host(rstd), t, None, None, 1e-5)


# -------------------------------------------------------------- gradients of a bias alone
@pytest.mark.parametrize("rows,cols,shift", [(300, 260, 0), (37, 4096, 0), (90, 33, 1), (0, 12, 0)])
def test_parameter_gradients_are_a_choice(tcx, rows, cols, shift):
    """params=True gives both sums without a weight (a norm with a bias alone), the same as with
    a weight of ones; params=False leaves them out (frozen parameters)."""
    x, _, w, b = norm_case(rows, cols, False)
    xd, wd, bd = dev(x, shift), dev(w), dev(b)
    dy = dev(np.random.default_rng(rows).normal(size=x.shape).astype(np.float32), shift)
    y, total, mean, rstd = tcx.layernorm_forward(xd, None, bd)
    ones = torch.ones(cols, device="cuda")
    want = tcx.layernorm_backward(dy, total, mean, rstd, ones)
    got = tcx.layernorm_backward(dy, total, mean, rstd, params=True)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    hat = (x.astype(np.float64) - host(mean)[:, None]) * host(rstd)[:, None]
    d = host(dy).astype(np.float64)
    within(host(got[2]), (d * hat).sum(0), (rows + 8) * U * np.abs(d * hat).sum(0), "dweight")
    within(host(got[3]), d.sum(0), (rows + 8) * U * np.abs(d).sum(0), "dbias")
    none = tcx.layernorm_backward(dy, total, mean, rstd)
    assert none[2] is None and none[3] is None and torch.equal(none[0], got[0])
    frozen = tcx.layernorm_backward(dy, total, mean, rstd, wd, params=False)
    with_them = tcx.layernorm_backward(dy, total, mean, rstd, wd)
    assert frozen[2] is None and frozen[3] is None and torch.equal(frozen[0], with_them[0])
    assert with_them[2] is not None and with_them[3] is not None
    with pytest.raises(TypeError, match="params"):
        tcx.layernorm_backward(dy, total, mean, rstd, wd, params=1)


# ---------------------------------------------------------------------------- large gates
@pytest.mark.parametrize("batch,time,channels", [(2, 512, 33), (1, 700, 128), (400, 128, 512), (300, 256, 32)])
@pytest.mark.parametrize("sign", [1, -1])
def test_recurrence_gates_of_the_largest_products(tcx, batch, time, channels, sign):
    """128 gates of 1.99 in a row, in one chunk or across two, whose product (1.8e38) a float32
    just holds; the states around them are tiny. h, dx and dinitial (a gate's gradient is a
    product of two such numbers, and leaves float32's range)."""
    gate, x, init, dh, dstate = recurrence_case(batch, time, channels, "decay", seed=11)
    gate *= np.float32(0.5)
    first = (time - 128) // 256 * 128  # a chunk's first step forward, within two backward
    gate[:, first:first + 128, ::2] = sign * np.float32(1.99)
    gate[:, (time - 128) // 2:(time - 128) // 2 + 128, 1::2] = sign * np.float32(1.99)
    x, init, dh, dstate = (v * np.float32(1e-25) for v in (x, init, dh, dstate))
    a, kappa, every = gate.astype(np.float64), roundings(gate, "decay"), np.ones((batch, time), bool)
    want, bound = scan(a, x.astype(np.float64), init, every, kappa)
    h, state = tcx.gated_recurrence(dev(gate), dev(x), dev(init))
    within(host(h), want, bound, "h")
    within(host(state), want[:, -1], bound[:, -1], "state")
    _, dx, dinit = tcx.gated_recurrence_backward(dev(dh), dev(gate), None, h, dev(init), dstate=dev(dstate))
    back, d = slice(None, None, -1), dh.astype(np.float64)
    c, off = (v[:, back] for v in scan(a[:, back], (a * d)[:, back], dstate, every, kappa))
    after = np.concatenate([c[:, 1:], dstate[:, None].astype(np.float64)], 1)
    off_after = np.concatenate([off[:, 1:], np.zeros((batch, 1, channels))], 1)
    within(host(dx), d + after, off_after + 2 * U * (np.abs(d) + np.abs(after)), "dx")
    within(host(dinit), c[:, 0], off[:, 0] + U * np.abs(c[:, 0]), "dinitial")


# ------------------------------------------------- sequences in buffers at any address
@pytest.mark.parametrize("form", ["decay", "sigmoid"])
@pytest.mark.parametrize("batch,time,channels,shift", [(250, 140, 21, 1), (1, 5000, 40, 1), (300, 300, 32, 2),
                                                       (5, 1700, 33, 3), (700, 100, 301, 1), (2, 40, 64, 1)])
def test_sequences_at_any_address(tcx, form, batch, time, channels, shift):
    """Whole chains to a block, a walk back over more than 8 chunks, a thread to a channel, with
    lengths that end anywhere, none, or past the end."""
    gate, x, init, dh, dstate = recurrence_case(batch, time, channels, form, seed=12)
    lengths = np.random.default_rng(time).integers(-1, time + 2, batch)
    lengths[:1] = time - 1
    pad = ~live_steps(batch, time, lengths)
    gate[pad], x[pad] = np.nan, np.inf
    check_recurrence(tcx, gate, x, init, dh, dstate, form, lengths, shift=shift)
    h, _ = tcx.gated_recurrence(dev(gate, shift), dev(x, shift), dev(init, shift), form=form,
                                lengths=dev(lengths.astype(np.int32)))
    h = host(h)
    for b, n in enumerate(np.clip(lengths, 0, time)):
        assert (h[b, n:] == (h[b, n - 1] if n else init[b])).all()


# --------------------------------------------------------------- NaN in front of a norm
@pytest.mark.parametrize("rows,cols,shift", [(40, 36, 0), (12, 1000, 0), (9, 4099, 0), (7, 10000, 0), (5, 20000, 0),
                                             (6, 100, 1)])
def test_norm_of_rows_with_nan_under_dropout(tcx, rows, cols, shift):
    """A NaN or an infinity makes its row NaN where it is kept and nothing where it is dropped."""
    p, seed = 0.5, 31
    x, r, w, b = norm_case(rows, cols, True)
    keep = mask_at(x.shape, p, seed, 3)
    hit = [(i, [0, cols // 2, cols - 1][i % 3]) for i in range(0, rows, 2)]
    for i, c in hit:
        x[i, c] = [np.nan, np.inf, -np.inf][i % 3]
    bad = np.array([any(i == j and keep[i, c] for i, c in hit) for j in range(rows)])
    for res in (None, r):
        y, total, mean, rstd = tcx.layernorm_forward(dev(x, shift), dev(w), dev(b), p=p, seed=seed, offset=3,
                                                     residual=None if res is None else dev(res, shift))
        with np.errstate(invalid="ignore"):
            want = np.where(keep, x * scale_of(p), np.float32(0)).astype(np.float32)
        want = want if res is None else res + want
        assert np.isnan(host(y)[bad]).all()
        check_forward(host(y)[~bad], host(mean)[~bad], host(rstd)[~bad], want[~bad], w, b, 1e-5)


# ---------------------------------------------------------------- host threads and streams
def one_of_each(tcx, seed, cols):
    """Every operator once, from inputs of the seed; long rows, clusters and scans among them."""
    make = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=make, device="cuda")
    x, r, w = normal(61, cols), normal(61, cols), normal(cols)
    y, total, mean, rstd = tcx.layernorm_forward(x, w, w, residual=r, p=0.2, seed=seed)
    out = [tcx.dropout(x, 0.3, seed), y, total, mean, rstd, *tcx.layernorm_forward(x, w)[::2]]
    out += tcx.layernorm_backward(y, total, mean, rstd, w, dtotal=r, p=0.2, seed=seed)
    gate, xs, dh = (normal(2, 700, cols // 64) for _ in range(3))
    h, state = tcx.gated_recurrence(gate, xs, form="sigmoid")
    return out + [h, state, *tcx.gated_recurrence_backward(dh, gate, xs, h, form="sigmoid")[:2]]


def test_host_threads_on_streams_of_their_own(tcx):
    """Four threads at a time, each on a side stream, get what one gets on the usual stream."""
    cols = [520, 9001, 12288, 17000]
    got, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[i] = [one_of_each(tcx, 10 * i + j, cols[(i + j) % 4]) for j in range(8)]
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001 (a thread's failure is the test's)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in range(4):
        for j in range(8):
            want = one_of_each(tcx, 10 * i + j, cols[(i + j) % 4])
            assert all(torch.equal(a, b) for a, b in zip(got[i][j], want)), (i, j)
