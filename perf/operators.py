"""The framework's large-language-model operators as measured cases: layer normalisation (forward, and forward with backward) and
the AdamW step over many tensors at once, with states in 8 bits or in 32 and optional clipping by the global gradient norm.

`run` computes a case in elementary torch operations, or, where `own` is true, through the framework's public entry points.
"""
import math
import random

import torch

own = False

KINDS = {"f32": torch.float32, "bf16": torch.bfloat16}
BETAS, LR, EPS, DECAY, STEP = (0.9, 0.999), 1e-4, 1e-3, 1e-2, 10    # the training configuration; STEP updates done before
BLOCK, MIN_8BIT = 256, 4096


# ---------------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------------
def _ln(name, train, dtype, rows, width, pad=0):
    return {"name": name, "op": "layer_norm", "train": train, "dtype": dtype, "rows": rows, "width": width, "pad": pad}


def _adamw(name, bits, dtype, tensors, params, clip):
    return {"name": name, "op": "adamw", "bits": bits, "dtype": dtype, "tensors": tensors, "params": params, "clip": clip}


def listed():
    return [
        # one 352x1216 image at 1/32 of its size, 512 channels, no gradient: the latency of a call
        _ln("ln_infer_1_image", False, "bf16", 418, 512),
        # a batch of 8 at 1/8, 128 channels, no gradient
        _ln("ln_infer_batch", False, "f32", 53504, 128),
        # rows that are a channel slice of a wider buffer, neither width nor stride a multiple of a vector
        _ln("ln_train_odd_slice", True, "f32", 4001, 667, 5),
        # a batch of 8 at 1/32: the widest feature map of the encoder
        _ln("ln_train_2208", True, "f32", 3344, 2208),
        # a batch of 8 at 1/16, 512 channels
        _ln("ln_train_512", True, "bf16", 13376, 512),
        # a batch of 8 at half size, 96 channels: long columns for the weight's gradient
        _ln("ln_train_half_res", True, "bf16", 856064, 96),
        # the parameters of one small head: the latency of a step
        _adamw("adamw8_head", 8, "f32", 6, 60000, 0.0),
        # as many tensors and parameters as the DenseNet161 model has
        _adamw("adamw8_densenet161", 8, "f32", 550, 47000688, 0.0),
        # as many as the ResNeXt101 model has, clipped
        _adamw("adamw8_resnext101_clip", 8, "f32", 382, 112765272, 1.0),
        # bf16 weights and gradients with 8-bit states, the MobileNetV2 model's counts
        _adamw("adamw8_bf16_clip", 8, "bf16", 224, 16338992, 1.0),
        # bf16 weights with 32-bit states
        _adamw("adamw32_bf16", 32, "bf16", 20, 20528688, 0.0),
        # f32 weights, 32-bit states, clipped: odd sizes
        _adamw("adamw32_clip", 32, "f32", 17, 5000001, 1.0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(("f32", "bf16"))
    if rng.random() < 0.55:
        width = _log(rng, 8, 8192)
        return {"op": "layer_norm", "train": rng.random() < 0.6, "dtype": dtype, "rows": _log(rng, 1, min(1000000, 80000000 // width)),
                "width": width, "pad": rng.choice((0, 0, 0, rng.randint(1, 64)))}
    bits = rng.choice((8, 8, 32))
    tensors = _log(rng, 1, 500 if bits == 8 else 20)
    return {"op": "adamw", "bits": bits, "dtype": dtype, "tensors": tensors,
            "params": max(tensors, _log(rng, 20000, 100000000 if bits == 8 else 60000000)), "clip": rng.choice((0.0, 1.0))}


def _sizes(case):
    """Lengths of the case's tensors: a few large ones hold most of the elements, many are short vectors."""
    rnd, n, total = random.Random(case["tensors"] * 1000003 + case["params"]), case["tensors"], case["params"]
    w = [math.exp(rnd.uniform(0.0, math.log(1e5))) for _ in range(n)]
    s = [max(1, int((total - n) * x / sum(w))) for x in w]
    s[s.index(max(s))] += total - sum(s)
    return s


def work(case):
    if case["op"] == "layer_norm":
        n, es = case["rows"] * case["width"], 2 if case["dtype"] == "bf16" else 4
        if case["train"]:
            return {"bytes": 4 * n * es + 16 * case["width"], "flops": 20 * n}
        return {"bytes": 2 * n * es + 8 * case["width"], "flops": 8 * n}
    es = 2 if case["dtype"] == "bf16" else 4
    total = 0
    for n in _sizes(case):
        eight = case["bits"] == 8 and n >= MIN_8BIT
        # weights read and written, gradients read, states read and written; 8-bit states come back as the values they stand for, too
        total += n * (3 * es + (4 if eight else 16) + (8 if case["bits"] == 8 else 0))
    return {"bytes": total, "flops": 15 * case["params"]}


# ---------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------
class _State:
    pass


def _blocks(sizes, device):
    """Where the blocks of 256 consecutive elements of every tensor lie in the tensors' concatenation: the index of each element of each
    block (0 behind a tensor's end), whether it is one, and whether the block's tensor has 8-bit states."""
    first, length, eight, off = [], [], [], 0
    for n in sizes:
        for b in range(0, n, BLOCK):
            first.append(off + b)
            length.append(min(BLOCK, n - b))
            eight.append(n >= MIN_8BIT)
        off += n
    lane = torch.arange(BLOCK, device=device)
    index = torch.tensor(first, device=device)[:, None] + lane
    valid = lane < torch.tensor(length, device=device)[:, None]
    return torch.where(valid, index, torch.zeros_like(index)), valid, torch.tensor(eight, device=device)[:, None]


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    s, dt = _State(), KINDS[case["dtype"]]
    s.case = case

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)
    if case["op"] == "layer_norm":
        M, C = case["rows"], case["width"]
        buf = (randn(M, C + case["pad"]) * 1.5).to(dt)
        buf += randn(C + case["pad"]).to(dt)                             # every channel has a mean of its own
        s.x = buf[:, :C].detach().requires_grad_(case["train"])
        s.w = (1.0 + 0.2 * randn(C)).requires_grad_(case["train"])
        s.b = (0.1 * randn(C)).requires_grad_(case["train"])
        s.dy = (randn(M, C) * 1e-2).to(dt) if case["train"] else None
        return s
    sizes = _sizes(case)
    total = sum(sizes)
    s.sizes, s.step = sizes, STEP
    level = torch.repeat_interleave(torch.exp(randn(len(sizes)) * 1.5 - 6.0), torch.tensor(sizes, device=dev))     # every tensor has its own gradient level
    s.p = (randn(total) * 0.05).to(dt)
    s.g = (randn(total) * level).to(dt)
    s.g[(torch.arange(total, device=dev) % 4099) < 40] = 0                # parameters that get no gradient this time
    s.m = randn(total) * level * 0.3
    s.v = (randn(total) ** 2 + 0.01) * level ** 2
    half = (len(sizes) + 1) // 2                                            # two groups: the first decays its weights
    s.decay = torch.full((total,), 0.0, device=dev)
    s.decay[:sum(sizes[:half])] = DECAY
    if case["bits"] == 8:
        s.index, s.valid, s.eight = _blocks(sizes, dev)
        s.m = _held_in_8(s, s.m.double(), 448.0, -6).float()
        s.v = _held_in_8(s, s.v.double(), 61440.0, -14).float()
    if own:
        s.opt = _optimizer(s, half)
    return s


def _optimizer(s, half):
    """The handle that a training program keeps: parameters and gradients are views of two flat buffers, states come from a checkpoint."""
    from bts_amd.optim import FusedAdamW
    ps = [torch.nn.Parameter(t) for t in torch.split(s.p, s.sizes)]
    for p, g in zip(ps, torch.split(s.g, s.sizes)):
        p.grad = g
    groups = [{"params": ps[:half], "weight_decay": DECAY}]
    if ps[half:]:
        groups.append({"params": ps[half:], "weight_decay": 0.0})
    opt = FusedAdamW(groups, lr=LR, betas=BETAS, eps=EPS, state_bits=s.case["bits"], max_grad_norm=s.case["clip"] or None, min_8bit_size=MIN_8BIT)
    saved = opt.state_dict()
    at = torch.tensor(float(STEP))
    saved["state"] = {i: {"step": at, "exp_avg": m, "exp_avg_sq": v}
                      for i, (m, v) in enumerate(zip(torch.split(s.m, s.sizes), torch.split(s.v, s.sizes)))}
    opt.load_state_dict(saved)
    s.m = s.v = None
    s.params = ps
    return opt


# ---------------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------------
def run(s):
    if s.case["op"] == "layer_norm":
        return _run_layer_norm_own(s) if own else _run_layer_norm(s)
    return _run_adamw_own(s) if own else _run_adamw(s)


def _run_layer_norm_own(s):
    from bts_amd.norm import layer_norm
    if not s.case["train"]:
        with torch.no_grad():
            return layer_norm(s.x, s.w, s.b, 1e-5)
    y = layer_norm(s.x, s.w, s.b, 1e-5)
    return (y.detach(),) + torch.autograd.grad(y, (s.x, s.w, s.b), s.dy)


@torch.no_grad()
def _run_layer_norm(s):
    x, w = s.x.float(), s.w
    C = x.shape[1]
    xc = x - x.sum(1, keepdim=True) / C
    r = 1.0 / torch.sqrt((xc * xc).sum(1, keepdim=True) / C + 1e-5)
    xh = xc * r
    y = (xh * w + s.b).to(s.x.dtype)
    if not s.case["train"]:
        return y
    dy = s.dy.float()
    h = dy * w
    dx = r * (h - h.sum(1, keepdim=True) / C - xh * ((h * xh).sum(1, keepdim=True) / C))
    return y, dx.to(s.x.dtype), (dy * xh).sum(0), dy.sum(0)


def _run_adamw_own(s):
    s.opt.step()
    if s.case["bits"] == 8:
        out = (s.p,) + tuple(s.opt.moments(flat=True))
    else:
        out = (s.p, [s.opt.state[p]["exp_avg"] for p in s.params], [s.opt.state[p]["exp_avg_sq"] for p in s.params])
    return out + ((s.opt.grad_norm,) if s.case["clip"] else ())


def _power(e):
    """2^e in 64 bits for whole e."""
    return ((e + 1023) << 52).view(torch.float64)


def _held_in_8(s, x, largest, lowest):
    """`x` as 8-bit states hold it: in blocks, as numbers of four significant bits between 2^lowest (below it, multiples of 2^(lowest - 3))
    and `largest`, times a power of two 2^k, k >= -126 the smallest with which the block's largest magnitude still fits. Rounded to nearest,
    ties to even. Tensors that are too short for 8 bits keep 32."""
    b = torch.where(s.valid, x[s.index], torch.zeros((), dtype=torch.float64, device=x.device))
    top = b.abs().amax(1, keepdim=True)
    e = (top.view(torch.int64) >> 52) - 1023
    four = torch.round(top * _power(3 - e.clamp_min(-900))) * _power(e.clamp_min(-900) - 3)        # the largest magnitude in four bits
    span = int(math.floor(math.log2(largest)))
    e4 = (four.view(torch.int64) >> 52) - 1023
    k = (e4 - span + (four * _power(span - e4.clamp_min(-900)) > largest).long()).clamp_min(-126)
    e = (b.abs().view(torch.int64) >> 52) - 1023
    unit = torch.maximum(e, k + lowest) - 3                                                            # a step of the numbers around each value
    q = torch.round(b * _power(-unit)) * _power(unit)
    if lowest == -14:                                                                                   # second moments: above zero stays above zero
        q = torch.where((b > 0) & (q == 0), _power(k + lowest - 3), q)
    q = torch.where(s.eight, q, b)
    out = torch.empty_like(x)
    out[s.index[s.valid]] = q[s.valid]
    return out


def _run_adamw(s):
    b1, b2 = BETAS
    s.step += 1
    wide = torch.float64 if s.case["bits"] == 8 else torch.float32      # values next to a border of their 8-bit form are decided in 64 bits
    g, more = s.g.to(wide), ()
    if s.case["clip"]:
        norm = torch.sqrt((s.g.double() * s.g.double()).sum())
        g = g * torch.clamp(s.case["clip"] / (norm + 1e-6), max=1.0).to(wide)
        more = (norm.float(),)
    m = b1 * s.m.to(wide) + (1 - b1) * g
    v = b2 * s.v.to(wide) + (1 - b2) * g * g
    step = LR / (1 - b1 ** s.step)
    p = s.p.to(wide) * (1 - LR * s.decay.to(wide)) - step * m / (torch.sqrt(v) / math.sqrt(1 - b2 ** s.step) + EPS)
    s.p.copy_(p)
    if s.case["bits"] == 8:
        s.m = _held_in_8(s, m, 448.0, -6).float()
        s.v = _held_in_8(s, v, 61440.0, -14).float()
        return (s.p, s.m, s.v) + more
    s.m, s.v = m, v
    return (s.p, list(torch.split(m, s.sizes)), list(torch.split(v, s.sizes))) + more


# ---------------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------
def _numbers(mantissa_steps, lowest, largest):
    """Every number >= 0 of an 8-bit form: `mantissa_steps` to a power of two, from 2^lowest (even steps below it) to `largest`."""
    got, unit = [i * 2.0 ** lowest / mantissa_steps for i in range(mantissa_steps)], 2.0 ** lowest
    while unit <= largest:
        got += [unit * (1 + i / mantissa_steps) for i in range(mantissa_steps) if unit * (1 + i / mantissa_steps) <= largest]
        unit *= 2
    return torch.tensor(got, dtype=torch.float64)


def _nearest(x, largest, lowest, limit, keep_above_zero):
    """One tensor in its 8-bit form by looking up the nearest of all its numbers. `limit`: what still rounds to `largest`."""
    n = x.numel()
    b = torch.cat((x, x.new_zeros(-n % BLOCK))).view(-1, BLOCK)
    top = b.abs().max(1, keepdim=True).values
    k = torch.full_like(top, -126.0)
    some = top > 0
    guess = torch.ceil(torch.log2(torch.where(some, top, torch.ones_like(top)) / limit))
    twos = torch.tensor([2.0 ** i for i in range(-300, 301)], dtype=torch.float64, device=x.device)      # pow() on a GPU may be a bit off
    for d in (1, 0, -1, -2):                                                   # the smallest of these with which the block fits
        at = top * twos[(300 - (guess + d)).long().clamp(0, 600)]
        k = torch.where(some & ((at <= limit) if largest == 448.0 else (at < limit)), (guess + d).clamp_min(-126.0), k)
    scale = twos[(k + 300).long()]
    table = _numbers(8, lowest, largest).to(x.device)
    a = (b.abs() / scale).clamp_max(largest)
    between = (table[1:] + table[:-1]) / 2
    code = torch.bucketize(a, between)
    code = code + ((code % 2 == 1) & (a == between[code.clamp_max(between.numel() - 1)])).long()       # ties to the even code
    if keep_above_zero:
        code = torch.where(a > 0, code.clamp_min(1), code)
    return (torch.sign(b) * table[code] * scale).view(-1)[:n]


@torch.no_grad()
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "layer_norm":
        x, w, b = s.x.double(), s.w.double(), s.b.double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        std = torch.sqrt(var + 1e-5)
        n = (x - mean) / std
        y = torch.addcmul(b, n, w)
        if not case["train"]:
            return y
        dy = s.dy.double()
        n_w = dy * w
        dx = (n_w - n_w.mean(1, keepdim=True) - n * (n_w * n).mean(1, keepdim=True)) / std
        return y, dx, torch.einsum("mc,mc->c", dy, n), dy.sum(0)
    b1, b2 = BETAS
    t, scale, norm = STEP + 1, 1.0, None
    if case["clip"]:
        norm = torch.linalg.vector_norm(s.g, dtype=torch.float64).item()
        scale = min(1.0, case["clip"] / (norm + 1e-6))
    ps, ms, vs, half, off = [], [], [], (len(s.sizes) + 1) // 2, 0
    for i, n in enumerate(s.sizes):
        p, g, m, v = (a[off:off + n].double() for a in (s.p, s.g, s.m, s.v))
        off += n
        g = g * scale
        m = torch.add(m * b1, g, alpha=1 - b1)
        v = torch.addcmul(v * b2, g, g, value=1 - b2)
        ps.append(p - LR * (DECAY if i < half else 0.0) * p - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS))
        if case["bits"] == 8 and n >= MIN_8BIT:
            m, v = _nearest(m, 448.0, -6, 464.0, False), _nearest(v, 61440.0, -14, 63488.0, True)
        ms.append(m)
        vs.append(v)
    if case["bits"] == 8:
        ms, vs = torch.cat(ms), torch.cat(vs)
    return (torch.cat(ps), ms, vs) + ((torch.tensor(norm, dtype=torch.float64),) if case["clip"] else ())
