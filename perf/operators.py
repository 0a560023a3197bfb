"""The training operators (dropout, layer norm, gated recurrence) at the sizes they are used at.

`own` chooses between the plain form (elementary torch operations in 32 bits) and the calls a
user makes of tensorcx_b200.ops; `exact` gives the same outputs from the definitions in 64 bits.
Everything is float32 as in the rest of the package; random numbers are the element's own place
in the counter-based stream of a seed (Philox4x32-10), so a mask is a function of (seed, place).
"""
import math

import numpy as np
import torch

own = False

# Element e of a seed's stream: word e % 4 of the Philox4x32-10 block e / 4, its upper 24 bits.
MULTIPLIERS = (0xD2511F53, 0xCD9E8D57)
WEYL = (0x9E3779B9, 0xBB67AE85)
LOW = 0xFFFFFFFF


def listed():
    return [
        # activations of a small hidden layer (256 rows of 512): bound by the call itself
        dict(name="dropout_small", op="dropout", rows=256, cols=512, p=0.1, offset=0, residual=False),
        # the residual branch of a large batch
        dict(name="dropout_residual", op="dropout", rows=16384, cols=4096, p=0.1, offset=0, residual=True),
        # the gradient of an odd-sized activation that starts inside a block of the stream, past 32 bits
        dict(name="dropout_backward_odd", op="dropout_backward", rows=4001, cols=1023, p=0.25, offset=(1 << 33) + 7),
        # the norm in front of a small layer, statistics kept for the backward pass
        dict(name="norm_small", op="norm", rows=256, cols=512, p=0.0, offset=0, residual=False),
        # dropout, residual addition and norm of a large batch in one call
        dict(name="norm_residual", op="norm", rows=16384, cols=4096, p=0.1, offset=0, residual=True),
        # the norm's gradient at the benchmark's row shape, with the weight's and the bias's
        dict(name="norm_backward", op="norm_backward", rows=16384, cols=4096, p=0.0, offset=0, residual=False),
        # the same through dropout and the residual branch, odd rows and columns
        dict(name="norm_backward_odd", op="norm_backward", rows=8191, cols=1001, p=0.1, offset=5, residual=True),
        # few long rows
        dict(name="norm_backward_wide", op="norm_backward", rows=2048, cols=32768, p=0.0, offset=0, residual=False),
        # one token for each of 256 running sequences
        dict(name="recurrence_token", op="recurrence", batch=256, time=1, channels=4096, form="sigmoid", ragged=False),
        # one long sequence: the scan over time is all the parallelism there is
        dict(name="recurrence_long", op="recurrence", batch=1, time=65536, channels=1024, form="decay", ragged=False),
        # a training step's gradient over two long sequences
        dict(name="recurrence_backward", op="recurrence_backward", batch=2, time=16384, channels=2048, form="sigmoid",
             ragged=False),
        # a padded batch of short sequences, odd in every direction
        dict(name="recurrence_backward_ragged", op="recurrence_backward", batch=7, time=1777, channels=1001,
             form="decay", ragged=True),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    def size(low, high):
        n = spread(low, high)
        return n if rng.random() < 0.5 else max(low, n // 16 * 16)

    op = rng.choice(["dropout", "dropout_backward", "norm", "norm_backward", "recurrence", "recurrence_backward"])
    if op.startswith("recurrence"):
        channels = size(32, 8192)
        time = 1 if op == "recurrence" and rng.random() < 0.25 else spread(2, 65536)
        batch = spread(1, max(1, min(256, (1 << 26) // (channels * time))))
        time = min(time, max(1, (1 << 26) // (channels * batch)))
        return dict(op=op, batch=batch, time=time, channels=channels, form=rng.choice(["decay", "sigmoid"]),
                    ragged=rng.random() < 0.4)
    cols = size(32, 32768)
    rows = spread(1, max(1, min(65536, (1 << 26) // cols)))
    offset = rng.choice([0, rows * cols, rng.randrange(1 << 20), (1 << 32) + rng.randrange(1 << 20)])
    if op == "dropout_backward":
        return dict(op=op, rows=rows, cols=cols, p=rng.choice([0.05, 0.1, 0.25, 0.5]), offset=offset)
    residual = rng.random() < 0.5
    p = rng.choice([0.05, 0.1, 0.25, 0.5]) if residual or op == "dropout" else 0.0
    return dict(op=op, rows=rows, cols=cols, p=p, offset=offset if p else 0, residual=residual)


def work(case):
    if case["op"].startswith("recurrence"):
        edge = case["batch"] * case["channels"]
        n = edge * case["time"]
        ragged = 4 * case["batch"] if case["ragged"] else 0
        if case["op"] == "recurrence":  # gate, x, h; the state before and (beyond one token, where it is h) after
            return dict(bytes=12 * n + 4 * edge * (2 if case["time"] > 1 else 1) + ragged,
                        flops=(2 if case["form"] == "decay" else 6) * n)
        # dh, gate, h (and x), dgate, dx; both states and their gradients
        return dict(bytes=(20 if case["form"] == "decay" else 24) * n + 12 * edge + ragged,
                    flops=(3 if case["form"] == "decay" else 9) * n)
    n = case["rows"] * case["cols"]
    if case["op"] == "dropout":
        return dict(bytes=(12 if case["residual"] else 8) * n, flops=(2 if case["residual"] else 1) * n)
    if case["op"] == "dropout_backward":
        return dict(bytes=8 * n, flops=n)
    ends = 8 * case["rows"]
    if case["op"] == "norm":  # x (and residual), y (and total), statistics, weight and bias
        return dict(bytes=(16 if case["residual"] else 8) * n + ends + 8 * case["cols"], flops=8 * n)
    # dy, total (and dtotal), the gradient of total (and of x), statistics, weight and both its gradients
    return dict(bytes=(20 if case["residual"] else 12) * n + ends + 12 * case["cols"], flops=14 * n)


def prepare(case, seed):
    make = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=make, device="cuda")

    def uniform(low, high, *shape):
        return torch.rand(shape, generator=make, device="cuda") * (high - low) + low

    s = dict(case=case, seed=(seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 64))
    if case["op"].startswith("recurrence"):
        b, t, d = case["batch"], case["time"], case["channels"]
        # decays between fast and slow forgetting; gate logits around a slow one
        s["gate"] = uniform(0.8, 0.9995, b, t, d) if case["form"] == "decay" else normal(b, t, d) * 1.5 + 1.5
        s["x"], s["initial"] = normal(b, t, d), normal(b, d)
        s["lengths"] = None
        if case["ragged"]:
            s["lengths"] = torch.randint(0, t + 1, (b,), generator=make, device="cuda", dtype=torch.int32)
        if case["op"] == "recurrence_backward":
            s["dh"], s["dstate"] = normal(b, t, d), normal(b, d)
            s["h"] = plain_recurrence(s["gate"], s["x"], s["initial"], case["form"], s["lengths"])[0]
        return s
    r, c = case["rows"], case["cols"]
    if case["op"] == "dropout_backward":
        s["dy"] = normal(r, c)
        return s
    if case["op"] == "dropout":
        s["x"] = normal(r, c)
        s["residual"] = normal(r, c) if case["residual"] else None
        return s
    # rows of N(0, 3) about a level of their own, weights about one, small biases
    s["weight"], s["bias"] = uniform(0.5, 1.5, c), normal(c) * 0.1
    s["x"] = normal(r, c) * 3 + normal(r, 1)
    if case["op"] == "norm":
        s["residual"] = normal(r, c) if case["residual"] else None
        return s
    s["total"] = s.pop("x")
    mean = s["total"].mean(1, dtype=torch.float64)
    s["mean"] = mean.float()
    s["rstd"] = ((s["total"].square().mean(1, dtype=torch.float64) - mean * mean) + 1e-5).rsqrt().float()
    s["dy"] = normal(r, c)
    s["dtotal"] = normal(r, c) if case["residual"] else None
    return s


def run(s):
    case = s["case"]
    if own:
        from tensorcx_b200 import ops
        if case["op"] == "dropout":
            return ops.dropout(s["x"], case["p"], s["seed"], offset=case["offset"], residual=s["residual"])
        if case["op"] == "dropout_backward":
            return ops.dropout_backward(s["dy"], case["p"], s["seed"], offset=case["offset"])
        if case["op"] == "norm":
            y, total, mean, rstd = ops.layernorm_forward(
                s["x"], s["weight"], s["bias"], residual=s["residual"], p=case["p"], seed=s["seed"],
                offset=case["offset"])
            return dict(y=y, total=total, mean=mean, rstd=rstd) if case["residual"] else dict(y=y, mean=mean, rstd=rstd)
        if case["op"] == "norm_backward":
            dx, dresidual, dweight, dbias = ops.layernorm_backward(
                s["dy"], s["total"], s["mean"], s["rstd"], s["weight"], dtotal=s["dtotal"], p=case["p"],
                seed=s["seed"], offset=case["offset"])
            out = dict(dx=dx, dweight=dweight, dbias=dbias)
            return dict(out, dresidual=dresidual) if case["residual"] else out
        if case["op"] == "recurrence":
            h, state = ops.gated_recurrence(s["gate"], s["x"], s["initial"], form=case["form"], lengths=s["lengths"])
            return dict(h=h, state=state)
        dgate, dx, dinitial = ops.gated_recurrence_backward(
            s["dh"], s["gate"], s["x"], s["h"], s["initial"], form=case["form"], lengths=s["lengths"],
            dstate=s["dstate"])
        return dict(dgate=dgate, dx=dx, dinitial=dinitial)
    if case["op"] == "dropout":
        return plain_dropout(s["x"], case["p"], s["seed"], case["offset"], s["residual"])
    if case["op"] == "dropout_backward":
        return plain_dropout(s["dy"], case["p"], s["seed"], case["offset"], None)
    if case["op"] == "norm":
        total = s["x"] if not case["residual"] else plain_dropout(s["x"], case["p"], s["seed"], case["offset"],
                                                                  s["residual"])
        mean = total.sum(1, keepdim=True) / total.shape[1]
        centred = total - mean
        rstd = 1 / torch.sqrt((centred * centred).sum(1, keepdim=True) / total.shape[1] + 1e-5)
        y = centred * rstd * s["weight"] + s["bias"]
        out = dict(y=y, mean=mean[:, 0], rstd=rstd[:, 0])
        return dict(out, total=total) if case["residual"] else out
    if case["op"] == "norm_backward":
        normed = (s["total"] - s["mean"][:, None]) * s["rstd"][:, None]
        scaled = s["dy"] * s["weight"]
        n = normed.shape[1]
        inner = (scaled * normed).sum(1, keepdim=True) / n
        dtotal = s["rstd"][:, None] * (scaled - scaled.sum(1, keepdim=True) / n - normed * inner)
        out = dict(dweight=(s["dy"] * normed).sum(0), dbias=s["dy"].sum(0))
        if not case["residual"]:
            return dict(out, dx=dtotal)
        dtotal = dtotal + s["dtotal"]
        return dict(out, dresidual=dtotal, dx=plain_dropout(dtotal, case["p"], s["seed"], case["offset"], None))
    if case["op"] == "recurrence":
        h, state = plain_recurrence(s["gate"], s["x"], s["initial"], case["form"], s["lengths"])
        return dict(h=h, state=state)
    return plain_recurrence_backward(s, case["form"])


def plain_uniform(seed, offset, count, device):
    """Elements [offset, offset + count) of the seed's uniform stream, by 64-bit integer operations."""
    first = offset // 4
    block = torch.arange(first, (offset + count + 3) // 4, device=device, dtype=torch.int64)
    k0, k1 = seed & LOW, seed >> 32

    def multiply(m, v):  # upper and lower half of a 32 x 32-bit product (it wraps within 64 bits)
        product = v * m
        return (product >> 32) & LOW, product & LOW

    def round_(x0, x1, x2, x3, r):
        high0, low0 = multiply(MULTIPLIERS[0], x0)
        high1, low1 = multiply(MULTIPLIERS[1], x2)
        return (high1 ^ x1 ^ ((k0 + r * WEYL[0]) & LOW), low1, high0 ^ x3 ^ ((k1 + r * WEYL[1]) & LOW), low0)

    x = (block & LOW, block >> 32, torch.zeros_like(block), torch.zeros_like(block))
    x = round_(*round_(*round_(*round_(*round_(*x, 0), 1), 2), 3), 4)
    x = round_(*round_(*round_(*round_(*round_(*x, 5), 6), 7), 8), 9)
    words = torch.stack(x, 1).reshape(-1)[offset - 4 * first:offset - 4 * first + count]
    return (words >> 8).to(torch.float32) * 2.0**-24


def plain_dropout(x, p, seed, offset, residual):
    keep = plain_uniform(seed, offset, x.numel(), x.device).view(x.shape) >= p
    y = torch.where(keep, x * (1 / (1 - p)), 0.0)
    return y if residual is None else residual + y


def inside(lengths, time, device):
    """[batch, time, 1] truth values: the steps that a sequence has."""
    return (torch.arange(time, device=device)[None, :] < lengths[:, None])[:, :, None]


def plain_scan(a, b):
    """All prefixes of h = a h + b over axis 1 from h = 0, and the prefixes' products, by doubling."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return a, b


def plain_recurrence(gate, x, initial, form, lengths):
    a = gate if form == "decay" else 1 / (1 + torch.exp(-gate))
    b = x if form == "decay" else x / (1 + torch.exp(gate))
    if lengths is not None:
        there = inside(lengths, gate.shape[1], gate.device)
        a, b = torch.where(there, a, 1.0), torch.where(there, b, 0.0)
    products, h = plain_scan(a, b)
    h = h + products * initial[:, None]
    return h, h[:, -1].clone()


def plain_recurrence_backward(s, form):
    gate, x, h = s["gate"], s["x"], s["h"]
    before = torch.cat([s["initial"][:, None], h[:, :-1]], 1)
    a = gate if form == "decay" else 1 / (1 + torch.exp(-gate))
    if s["lengths"] is not None:
        there = inside(s["lengths"], gate.shape[1], gate.device)
        a = torch.where(there, a, 1.0)
    # c_t = a_t (c_(t+1) + dh_t) runs from the last step to the first
    products, c = plain_scan(a.flip(1), (a * s["dh"]).flip(1))
    c = (c + products * s["dstate"][:, None]).flip(1)
    g = s["dh"] + torch.cat([c[:, 1:], s["dstate"][:, None]], 1)
    if form == "decay":
        dgate, dx = g * before, g
    else:
        rest = 1 / (1 + torch.exp(gate))
        dgate, dx = g * (before - x) * a * rest, g * rest
    if s["lengths"] is not None:
        dgate, dx = torch.where(there, dgate, 0.0), torch.where(there, dx, 0.0)
    return dict(dgate=dgate, dx=dx, dinitial=c[:, 0].clone())


def exact_keep(seed, offset, shape, p):
    """Which elements a dropout keeps, from the stream's definition (64-bit host arithmetic)."""
    count = int(np.prod(shape))
    start = offset // 4
    blocks = np.arange(start, (offset + count - 1) // 4 + 1, dtype=np.uint64)
    half, low = np.uint64(32), np.uint64(LOW)
    c = [blocks & low, blocks >> half, np.zeros_like(blocks), np.zeros_like(blocks)]
    key = [seed % 2**32, seed // 2**32]
    for _ in range(10):
        left, right = c[0] * np.uint64(MULTIPLIERS[0]), c[2] * np.uint64(MULTIPLIERS[1])
        c = [(right >> half) ^ c[1] ^ np.uint64(key[0]), right & low, (left >> half) ^ c[3] ^ np.uint64(key[1]),
             left & low]
        key = [(k + w) % 2**32 for k, w in zip(key, WEYL)]
    bits = np.stack([w >> np.uint64(8) for w in c], axis=1).ravel()[offset % 4:offset % 4 + count]
    return torch.from_numpy((bits.astype(np.float64) / 2**24 >= p).reshape(shape))


def exact_dropout(case, s, v):
    keep = exact_keep(s["seed"], case["offset"], tuple(v.shape), case["p"]).to(v.device)
    return v.double().masked_fill(~keep, 0).div(1 - case["p"])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "dropout":
        y = exact_dropout(case, s, s["x"])
        return y if s["residual"] is None else y + s["residual"].double()
    if case["op"] == "dropout_backward":
        return exact_dropout(case, s, s["dy"])
    if case["op"] == "norm":
        total = s["x"].double()
        if case["residual"]:
            total = exact_dropout(case, s, s["x"]) + s["residual"].double()
        variance, mean = torch.var_mean(total, 1, correction=0)
        rstd = (variance + 1e-5) ** -0.5
        y = torch.addcmul(s["bias"].double(), (total - mean[:, None]) * rstd[:, None], s["weight"].double())
        out = dict(y=y, mean=mean, rstd=rstd)
        return dict(out, total=total) if case["residual"] else out
    if case["op"] == "norm_backward":
        dy, r = s["dy"].double(), s["rstd"].double()[:, None]
        hat = (s["total"].double() - s["mean"].double()[:, None]) * r
        g = dy * s["weight"].double()
        d = r * (g - g.mean(1, keepdim=True) - hat * torch.mean(g * hat, 1, keepdim=True))
        out = dict(dweight=torch.einsum("rc,rc->c", dy, hat), dbias=dy.sum(0))
        if not case["residual"]:
            return dict(out, dx=d)
        d = d + s["dtotal"].double()
        return dict(out, dresidual=d, dx=exact_dropout(case, s, d))
    # step by step through time, [time, batch, channels]
    last = case["time"]
    ends = s["lengths"].tolist() if case["ragged"] else [last] * case["batch"]
    live = torch.zeros(last, case["batch"], 1, dtype=torch.float64, device=s["gate"].device)
    for b, n in enumerate(ends):
        live[:n, b] = 1
    gate, x = s["gate"].double().transpose(0, 1), s["x"].double().transpose(0, 1)
    a, rest = (gate, torch.ones_like(gate)) if case["form"] == "decay" else (torch.sigmoid(gate), torch.sigmoid(-gate))
    keep = torch.lerp(torch.ones_like(a), a, live)
    if case["op"] == "recurrence":
        h, state = rest * x * live, s["initial"].double()
        for t in range(last):
            state = h[t].addcmul_(keep[t], state)
        return dict(h=h.transpose(0, 1).contiguous(), state=state.clone())
    dh, h = s["dh"].double().transpose(0, 1), s["h"].double().transpose(0, 1)
    before = torch.cat([s["initial"].double()[None], h[:-1]])
    total, c = dh.clone(), s["dstate"].double()
    for t in reversed(range(last)):
        c = total[t].add_(c) * keep[t]
    dx = total * rest * live
    dgate = total * before * live if case["form"] == "decay" else dx * a * (before - x)
    return dict(dgate=dgate.transpose(0, 1).contiguous(), dx=dx.transpose(0, 1).contiguous(), dinitial=c)
