"""The training operators where their arguments end: places of the random stream at 2^64, outputs
that a call without dropout need not have.

The masks are compared with the generator's definition in whole-number arithmetic on the host.
"""
import numpy as np
import pytest
import torch

from test_gpu_training import dev, host, norm_case, scale_of

pytestmark = pytest.mark.gpu


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
