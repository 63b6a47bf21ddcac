"""Layer normalisation (bts_amd.norm, ops.layer_norm_*) against the definition in 64 bits.

Tolerances, with u = 2^-24 (half a step of f32).  A row sum adds at most 32 elements per lane and then exchanges over at most 2^10
lanes: <= 42 additions, so the mean is off by <= 43 u A with A = mean |x|, and every centred value by that plus u |xc|.  Relative to
s = sqrt(var + eps) the normalised value xh is then off by <= 43 u A / s (its own centring) + |xh| (43 u A / s + 50 u) (variance:
centring twice under a square root, 42 additions halved by it; reciprocal, square root and two products), which TOL (1 + |xh|) with
TOL = 128 u (1 + A / s) covers with room to spare.  A result stored in bf16 adds half a step: 2^-8 of the value."""
import pytest
import torch

from bts_amd import ops
from bts_amd._lib import BtsAmdError
from bts_amd.norm import LayerNorm, LayerNorm2d, layer_norm

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


def plain(x, w, b, eps, dy=None):
    """Everything in 64 bits on the CPU, with the scales that the tolerances are made of."""
    x = x.detach().double().cpu()
    x = x.reshape(-1, x.shape[-1])
    one = torch.ones(x.shape[1], dtype=torch.float64)
    w = one if w is None else w.detach().double().cpu()
    b = one * 0 if b is None else b.detach().double().cpu()
    mu = x.mean(1, keepdim=True)
    s = ((x - mu).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (x - mu) / s
    tol = 128 * U * (1 + x.abs().mean(1, keepdim=True) / s) * (1 + xh.abs())         # of xh
    r = {"y": xh * w + b, "tol_y": tol * w.abs() + 2 * U * (xh * w).abs() + U * b.abs(), "mean": mu[:, 0], "rstd": 1 / s[:, 0]}
    if dy is not None:
        g = dy.detach().double().cpu().reshape(x.shape)
        h = g * w
        m1, m2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
        a1, a2 = h.abs().mean(1, keepdim=True), (h.abs() * (xh.abs() + tol / (128 * U))).mean(1, keepdim=True)
        r["dx"] = (h - m1 - xh * m2) / s
        # h, its two means (42 additions) and their products with xh, each with the relative error of rstd
        rel = 128 * U * (1 + x.abs().mean(1, keepdim=True) / s)
        r["tol_dx"] = (rel * (h.abs() + a1 + (1 + xh.abs()) * a2)) / s
        n = x.shape[0] + 64                                                          # additions of a column, one by one at the worst
        r["dw"], r["db"] = (g * xh).sum(0), g.sum(0)
        r["tol_dw"], r["tol_db"] = (g.abs() * tol).sum(0) + n * U * (g * xh).abs().sum(0), n * U * g.abs().sum(0)
    return r


def within(got, want, tol, what, half=U):
    got = got.detach().double().cpu().reshape(want.shape)
    assert torch.isfinite(got).all(), what
    bad = (got - want).abs() - tol - half * (want.abs() + tol)
    assert bad.max().item() <= 1e-30, "%s: off by %.3g more than the tolerance at %d" % (what, bad.max().item(), bad.argmax().item())


def make(M, C, dtype, seed, pad=0, offset=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    flat = torch.randn(M * (C + pad) + offset, generator=gen, device=DEV) * 1.7 + 0.3
    x = flat.to(dtype)[offset:].view(M, C + pad)[:, :C]
    w = 1 + 0.3 * torch.randn(C, generator=gen, device=DEV)
    b = 0.2 * torch.randn(C, generator=gen, device=DEV)
    dy = (torch.randn(M, C + pad, generator=gen, device=DEV) * 0.1).to(dtype)[:, :C]
    return x, w, b, dy


SHAPES = [(1, 1), (3, 2), (5, 3), (1, 7), (33, 8), (257, 16), (70, 17), (100, 33), (1000, 32), (513, 96), (66, 127), (9, 130), (418, 512), (31, 667), (40, 1024),
          (17, 1025), (700, 1401), (33, 1537), (300, 2208), (19, 2049), (600, 2600), (7, 4097), (5, 8192), (3, 16384), (4, 16381), (20000, 24), (5000, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C", SHAPES)
def test_forward_and_backward(M, C, dtype):
    x, w, b, dy = make(M, C, dtype, M * 31 + C)
    y, stats = ops.layer_norm_fwd(x, w, b, 1e-5, want_stats=True)
    dx, dw, db = ops.layer_norm_bwd(dy, x, stats, w)
    torch.cuda.synchronize()
    r = plain(x, w, b, 1e-5, dy)
    assert y.dtype == dx.dtype == dtype and y.is_contiguous() and dx.is_contiguous() and dw.dtype == db.dtype == torch.float32
    within(y, r["y"], r["tol_y"], "y", HALF[dtype])
    within(dx, r["dx"], r["tol_dx"], "dx", HALF[dtype])
    within(dw, r["dw"], r["tol_dw"], "dweight")
    within(db, r["db"], r["tol_db"], "dbias")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C,pad,offset", [(50, 16, 3, 1), (50, 17, 0, 1), (37, 96, 32, 5), (21, 667, 5, 3), (9, 2208, 1, 7), (5, 8191, 9, 1)])
def test_strided_rows_at_any_address(M, C, pad, offset, dtype):
    x, w, b, dy = make(M, C, dtype, 7, pad, offset)
    assert pad == 0 or not x.is_contiguous()
    y, stats = ops.layer_norm_fwd(x, w, b, 1e-5, want_stats=True)
    dx, dw, db = ops.layer_norm_bwd(dy, x, stats, w)
    r = plain(x, w, b, 1e-5, dy)
    within(y, r["y"], r["tol_y"], "y", HALF[dtype])
    within(dx, r["dx"], r["tol_dx"], "dx", HALF[dtype])
    within(dw, r["dw"], r["tol_dw"], "dweight")
    within(db, r["db"], r["tol_db"], "dbias")


def test_entry_points_write_only_their_rows():
    """Through the C entry with strided outputs: what lies between and behind the rows keeps its values."""
    import ctypes as C
    from bts_amd._lib import BTS_F32, call, stream_ptr
    M, N, S = 37, 45, 51
    x, w, b, dy = make(M, N, torch.float32, 3)
    x, dy = x.contiguous(), dy.contiguous()
    y, dx = torch.full((M + 2, S), 7.0, device=DEV), torch.full((M + 2, S), 7.0, device=DEV)
    stats = torch.full((2, M + 1), 7.0, device=DEV)
    p = lambda t: C.c_void_p(t.data_ptr())   # noqa: E731
    call("bts_layernorm_fwd", p(x), BTS_F32, N, p(y), S, M, N, p(w), p(b), 1e-5, p(stats[0]), p(stats[1]), stream_ptr())
    call("bts_layernorm_bwd", p(dy), N, p(x), N, p(dx), S, BTS_F32, M, N, p(w), p(stats[0]), p(stats[1]), C.c_void_p(0), C.c_void_p(0),
         C.c_void_p(0), stream_ptr())
    r = plain(x, w, b, 1e-5, dy)
    within(y[:M, :N].contiguous(), r["y"], r["tol_y"], "y")
    within(dx[:M, :N].contiguous(), r["dx"], r["tol_dx"], "dx")
    for t in (y, dx):
        assert (t[:, N:] == 7.0).all() and (t[M:] == 7.0).all()
    assert (stats[:, M:] == 7.0).all()


@pytest.mark.parametrize("want", [(True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, True, False)])
@pytest.mark.parametrize("C", [48, 2208])
def test_only_what_is_asked_for(C, want):
    x, w, b, dy = make(65, C, torch.float32, 11)
    _, stats = ops.layer_norm_fwd(x, w, b, 1e-5, want_stats=True)
    full = ops.layer_norm_bwd(dy, x, stats, w)
    part = ops.layer_norm_bwd(dy, x, stats, w, *want)
    for f, p, k in zip(full, part, want):
        assert (p is None) != k
        assert not k or torch.equal(f, p)


@pytest.mark.parametrize("w,b", [(True, False), (False, True), (False, False)])
def test_without_weight_or_bias(w, b):
    x, wt, bs, dy = make(129, 40, torch.float32, 5)
    wt, bs = wt if w else None, bs if b else None
    x.requires_grad_(True)
    y = layer_norm(x, wt, bs)
    (dx,) = torch.autograd.grad(y, x, dy)
    r = plain(x, wt, bs, 1e-5, dy)
    within(y, r["y"], r["tol_y"], "y")
    within(dx, r["dx"], r["tol_dx"], "dx")


def test_constant_rows_and_rows_far_from_zero():
    """Variance 0 gives y = bias; a mean of 1000 times the spread loses A / s of the tolerance and no more (no E[x^2] - mean^2)."""
    _, w, b, dy = make(4, 200, torch.float32, 9)
    x = torch.full((4, 200), 3.25, device=DEV)
    y, stats = ops.layer_norm_fwd(x, w, b, 1e-5, want_stats=True)
    assert torch.equal(y, b.expand(4, 200)) and torch.equal(stats[0], x[:, 0])
    x = 1000 + torch.randn(4, 200, device=DEV)
    y, stats = ops.layer_norm_fwd(x, w, b, 1e-5, want_stats=True)
    dx, _, _ = ops.layer_norm_bwd(dy, x, stats, w)
    r = plain(x, w, b, 1e-5, dy)
    within(y, r["y"], r["tol_y"], "y")
    within(dx, r["dx"], r["tol_dx"], "dx")


def test_nan_and_infinity_stay_in_their_rows():
    x, w, b, dy = make(300, 96, torch.float32, 13)
    clean = layer_norm(x, w, b)
    bad = x.clone()
    bad[7, 3], bad[100, 95], bad[299, 0] = float("nan"), float("inf"), -float("inf")
    y = layer_norm(bad, w, b)
    rows = torch.ones(300, dtype=torch.bool, device=DEV)
    rows[[7, 100, 299]] = False
    assert torch.equal(y[rows], clean[rows]) and torch.isnan(y[~rows]).all()


def test_no_rows():
    w, b = torch.ones(5, device=DEV), torch.zeros(5, device=DEV)
    x = torch.empty(0, 5, device=DEV, requires_grad=True)
    w.requires_grad_(True)
    y = layer_norm(x, w, b)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty(0, 5, device=DEV))
    assert y.shape == dx.shape == (0, 5) and torch.equal(dw, torch.zeros(5, device=DEV))


def test_sums_have_a_fixed_order():
    x, w, b, dy = make(30011, 96, torch.bfloat16, 17)
    _, stats = ops.layer_norm_fwd(x, w, b, 1e-5, want_stats=True)
    first = ops.layer_norm_bwd(dy, x, stats, w)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, ops.layer_norm_bwd(dy, x, stats, w)))


def test_autograd_against_formula_and_differences():
    """3-D input, broadcast output gradient; then L(x + h d) - L(x - h d) over 2 h with the kernel's own forward pass."""
    x, w, b, _ = make(6 * 7, 50, torch.float32, 19)
    x = x.reshape(6, 7, 50).clone().requires_grad_(True)
    w.requires_grad_(True)
    b.requires_grad_(True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y.square().sum(), (x, w, b))
    r = plain(x, w, b, 1e-5, 2 * y.detach())
    within(dx, r["dx"], r["tol_dx"], "dx")
    within(dw, r["dw"], r["tol_dw"], "dweight")
    within(db, r["db"], r["tol_db"], "dbias")
    gs = torch.autograd.grad(layer_norm(x, w, b).sum(), (x, w, b))                       # gradient of a sum: an expanded scalar
    assert torch.equal(gs[2], torch.full_like(b, 42.0))
    r = plain(x, w, b, 1e-5, torch.ones_like(x))
    within(gs[0], r["dx"], r["tol_dx"], "dx of a sum")

    def loss(x, w, b):
        with torch.no_grad():
            return layer_norm(x, w, b).double().square().sum().item()
    gen = torch.Generator(device=DEV).manual_seed(23)
    h = 2.0 ** -7
    for t, g, at in ((x, dx, 0), (w, dw, 1), (b, db, 2)):
        d = torch.randn(t.shape, generator=gen, device=DEV) * 0.5
        args = [x.detach(), w.detach(), b.detach()]
        lo, hi = list(args), list(args)
        lo[at], hi[at] = args[at] - h * d, args[at] + h * d
        diff = (loss(*hi) - loss(*lo)) / (2 * h)
        want = (g.double() * d.double()).sum().item()
        # third derivatives of the loss along d are O(|L|); y itself carries 2100 independent errors of ~1e-6 relative
        total = loss(*args)
        assert abs(diff - want) <= h * h * 4 * total + 1e-6 * total / h, (at, diff, want)


def test_modules_match_torch():
    torch.manual_seed(0)
    a, t = LayerNorm((3, 40), eps=1e-6).to(DEV), torch.nn.LayerNorm((3, 40), eps=1e-6).to(DEV)
    with torch.no_grad():
        t.weight.copy_(torch.rand(3, 40) + 0.5)
        t.bias.copy_(torch.randn(3, 40))
    assert list(a.state_dict()) == list(t.state_dict())
    a.load_state_dict(t.state_dict())
    x = torch.randn(11, 2, 3, 40, device=DEV)
    xa, xt = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    ya, yt = a(xa), t(xt)
    dy = torch.randn_like(yt)
    ya.backward(dy)
    yt.backward(dy)
    for p, q in ((ya, yt), (xa.grad, xt.grad), (a.weight.grad, t.weight.grad), (a.bias.grad, t.bias.grad)):
        assert p.shape == q.shape and (p - q).abs().max() <= 1e-5 * q.abs().max()
    with pytest.raises(BtsAmdError):
        a(torch.randn(11, 40, 3, device=DEV))


@pytest.mark.parametrize("layout", ["nchw", "channels_last", "slice"])
def test_layer_norm_2d(layout):
    torch.manual_seed(1)
    m = LayerNorm2d(24).to(DEV)
    with torch.no_grad():
        m.weight.copy_(torch.rand(24) + 0.5)
    x = torch.randn(2, 32, 5, 7, device=DEV)
    if layout != "nchw":
        x = x.contiguous(memory_format=torch.channels_last)
    x = (x[:, 4:28] if layout == "slice" else x[:, :24].contiguous(memory_format=torch.channels_last if layout != "nchw" else torch.contiguous_format))
    x = x.detach().requires_grad_(True)
    y = m(x)
    dy = torch.randn_like(y)
    y.backward(dy)
    assert y.shape == x.shape and y.is_contiguous(memory_format=torch.channels_last)
    rows = lambda t: t.detach().permute(0, 2, 3, 1).reshape(-1, 24)   # noqa: E731
    r = plain(rows(x), m.weight, m.bias, 1e-5, rows(dy))
    within(rows(y), r["y"], r["tol_y"], "y")
    within(rows(x.grad), r["dx"], r["tol_dx"], "dx")
    within(m.weight.grad, r["dw"], r["tol_dw"], "dweight")


def test_captured_pass_replays_on_new_inputs():
    """Forward and backward in one graph, replayed several times between eager work; the tensors have no eager graph alive."""
    x, w, b, dy = make(700, 96, torch.float32, 29)
    x, dy = x.contiguous(), dy.contiguous()

    def step():
        y, stats = ops.layer_norm_fwd(x, w, b, 1e-5, want_stats=True)
        return (y,) + ops.layer_norm_bwd(dy, x, stats, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        one = step()
    with torch.cuda.graph(g2):
        two = step()
    for i in range(4):
        x.copy_(torch.randn_like(x) * (i + 1))
        dy.copy_(torch.randn_like(dy))
        g1.replay()
        g2.replay()
        want = step()
        torch.cuda.synchronize()
        for o, t, v in zip(one, two, want):
            assert torch.equal(o, v) and torch.equal(t, v), i


def test_on_a_stream_of_its_own():
    x, w, b, dy = make(4001, 130, torch.bfloat16, 31)
    want = layer_norm(x, w, b)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late = x.clone().mul_(2)
        late.copy_(x)
        got = layer_norm(late, w, b)
    s.synchronize()
    assert torch.equal(got, want)


def test_two_threads_at_once():
    """Two host threads, a stream each, forward and backward: every result is the one that a thread alone gets."""
    import threading
    cases = [make(3001, 96, torch.float32, 41), make(777, 2208, torch.bfloat16, 43)]
    want, got, errors = [], [[], []], []
    for x, w, b, dy in cases:
        y, stats = ops.layer_norm_fwd(x, w, b, 1e-5, want_stats=True)
        want.append((y,) + ops.layer_norm_bwd(dy, x, stats, w))
    torch.cuda.synchronize()

    def work(i):
        try:
            x, w, b, dy = (t.detach().clone().requires_grad_(k < 3) for k, t in enumerate(cases[i]))
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(s):
                for _ in range(20):
                    y = layer_norm(x, w, b)
                    got[i] = (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)
            s.synchronize()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors, errors
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_offsets_beyond_32_bits():
    """2^31 + 6400 elements: the last rows come out like those of a short tensor, and the sums count every row."""
    C, tail = 64, 100
    M = 2 ** 31 // C + tail
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of free device memory")
    gen = torch.Generator(device=DEV).manual_seed(47)
    x = torch.zeros(M, C, dtype=torch.bfloat16, device=DEV)
    x[-tail:] = torch.randn(tail, C, generator=gen, device=DEV).to(torch.bfloat16)
    w, b = torch.rand(C, generator=gen, device=DEV) + 0.5, torch.randn(C, generator=gen, device=DEV)
    y, stats = ops.layer_norm_fwd(x, w, b, 1e-5, want_stats=True)
    short, sstats = ops.layer_norm_fwd(x[-tail:], w, b, 1e-5, want_stats=True)
    assert torch.equal(y[-tail:], short) and torch.equal(stats[:, -tail:], sstats) and torch.equal(y[:3], b.to(torch.bfloat16).expand(3, C))
    dy = y.zero_()
    dy[-tail:] = torch.randn(tail, C, generator=gen, device=DEV).to(torch.bfloat16)
    dy[0] = 1.0                                                             # a constant row: xh = 0, adds to the bias's gradient only
    dx, dw, db = ops.layer_norm_bwd(dy, x, stats, w)
    sdx, _, _ = ops.layer_norm_bwd(dy[-tail:], x[-tail:], sstats, w)
    assert torch.equal(dx[-tail:], sdx) and (dx[1000:2000] == 0).all()
    r = plain(x[-tail:], w, b, 1e-5, dy[-tail:])
    within(dw, r["dw"], r["tol_dw"], "dweight")
    within(db - 1.0, r["db"], r["tol_db"] + 200 * U, "dbias")


def test_refusals_on_the_device():
    x, w, b, dy = make(8, 16, torch.float32, 37)
    for args in ((x.half(), w, b), (x.double(), w, b), (x, w[:15], b), (x, w.bfloat16(), b), (x, w.cpu(), b), (x, w, b[:1]),
                 (torch.empty(2, ops.LN_MAX_C + 1, device=DEV), None, None), (torch.empty(4, 0, device=DEV), None, None)):
        with pytest.raises(BtsAmdError):
            layer_norm(*args)
    with pytest.raises(BtsAmdError):
        layer_norm(x, w, b, -1.0)
    with pytest.raises(BtsAmdError):
        ops.layer_norm_fwd(x.t(), None, None)
    _, stats = ops.layer_norm_fwd(x, w, b, want_stats=True)
    for args in ((dy[:7], x, stats, w), (dy.bfloat16(), x, stats, w), (dy, x, None, w), (dy, x, stats[:, :7], w), (dy, x, stats.double(), w),
                 (dy, x, stats, w[:3])):
        with pytest.raises(BtsAmdError):
            ops.layer_norm_bwd(*args)
    # gradients of gradients are refused, not wrong
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(layer_norm(x, w, b).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_tensor_hooks_may_change_the_layout(dtype):
    """save_on_cpu gives a channel slice back as a dense tensor: the gradients are those of the pass without hooks."""
    x, w, b, dy = make(401, 667, dtype, 53, pad=5)
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    want = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True), torch.autograd.graph.saved_tensors_hooks(torch.clone, lambda t: t)):
        with hooks:
            y = layer_norm(x, w, b)
        got = torch.autograd.grad(y, (x, w, b), dy)
        assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [1, 3, 7, 13, 30, 41, 100, 200, 257, 667, 1025, 2208, 2900, 4097, 8191, 9001, 16384])
def test_rows_of_equal_elements_are_centred_exactly(C, dtype):
    """Variance 0, whatever the value and the width.  Far from zero (|mean| > 4 sqrt(eps)) y is the bias and the mean is the value, bit for
    bit, and the weight's gradient is 0; below, and for the statistics of what is left there, the tolerances of any row hold."""
    values = torch.tensor([3.25, 1000.0, 1000.1, 30000.0, -0.1, 1.0 / 3, 65504.0, -1e6, 2.0 ** 20 + 0.3, 0.0, 1e-30, 1e-3, -0.01], device=DEV).to(dtype)
    M, far = values.numel(), 10
    _, w, b, dy = make(M, C, dtype, 61)
    x = values[:, None].expand(M, C).contiguous()
    y, stats = ops.layer_norm_fwd(x, w, b, 1e-5, want_stats=True)
    assert torch.equal(y[:far], b.to(dtype).expand(far, C)) and torch.equal(stats[0, :far], values[:far].float())
    assert ((stats[1].double() * 1e-5 ** 0.5 - 1).abs() <= 4 * U).all()                # root, reciprocal, eps in f32
    dx, dw, db = ops.layer_norm_bwd(dy, x, stats, w)
    r = plain(x, w, b, 1e-5, dy)
    within(y, r["y"], r["tol_y"], "y", HALF[dtype])
    within(dx, r["dx"], r["tol_dx"], "dx", HALF[dtype])
    within(db, r["db"], r["tol_db"], "dbias")
    _, dw, _ = ops.layer_norm_bwd(dy[:far], x[:far], stats[:, :far].contiguous(), w)
    assert (dw == 0).all()


@pytest.mark.parametrize("C", [41, 667, 2208, 9001])
def test_nearly_equal_elements_far_from_zero(C):
    """Rows at 1000 whose elements differ in the last bits: the spread is 2^-13 of sqrt(eps) and less, and what the kernel centres is exact,
    so the normalised values are good to a few roundings of their largest -- without the mean's own rounding, magnified."""
    gen = torch.Generator(device=DEV).manual_seed(67)
    steps = torch.randint(-3, 4, (50, C), generator=gen, device=DEV)
    x = (1000.0 + steps.double() * 2.0 ** -14).float()
    y, stats = ops.layer_norm_fwd(x, None, None, 1e-5, want_stats=True)
    x64 = x.double()
    xc = x64 - x64.mean(1, keepdim=True)
    want = xc / (xc.square().mean(1, keepdim=True) + 1e-5).sqrt()
    # elements and mean are multiples of 2^-14 below 2^10: a difference of them is exact, but for the mean's correction, which adds up at
    # most 42 times (u each) and is at most 43 u 1000 itself; root, reciprocal, product
    assert ((y.double() - want).abs() <= 50 * U * (want.abs() + 43 * U * 1000 / 1e-5 ** 0.5)).all()


# the kernel variants that SHAPES leaves out, and rows of odd width of which a block walks several (the next one is fetched ahead)
F, B = torch.float32, torch.bfloat16
MORE = [(F, 70, 4), (F, 65, 13), (F, 30, 200), (F, 31, 259), (F, 21, 640), (F, 19, 900), (F, 17, 1536), (F, 5, 9001), (F, 4, 12288), (B, 65, 11), (B, 30, 200),
        (B, 31, 301), (B, 17, 1280), (B, 13, 1800), (B, 11, 2901), (B, 9, 3333), (B, 6, 4096),
        (F, 9001, 201), (F, 9001, 301), (F, 9001, 667), (F, 5000, 1001), (F, 2100, 1401), (F, 1500, 2207), (F, 800, 8191), (F, 600, 9001), (F, 600, 16381),
        (B, 40001, 41), (B, 9001, 301), (B, 9001, 667), (B, 3000, 1401), (B, 2500, 1801), (B, 2100, 2207), (B, 1500, 2901), (B, 1500, 3333), (B, 800, 8191), (B, 600, 9001)]


@pytest.mark.parametrize("dtype,M,C", MORE)
def test_forward_and_backward_of_every_variant(dtype, M, C):
    x, w, b, dy = make(M, C, dtype, M * 37 + C)
    y, stats = ops.layer_norm_fwd(x, w, b, 1e-5, want_stats=True)
    dx, dw, db = ops.layer_norm_bwd(dy, x, stats, w)
    r = plain(x, w, b, 1e-5, dy)
    within(y, r["y"], r["tol_y"], "y", HALF[dtype])
    within(dx, r["dx"], r["tol_dx"], "dx", HALF[dtype])
    within(dw, r["dw"], r["tol_dw"], "dweight")
    within(db, r["db"], r["tol_db"], "dbias")
    dx_only, _, _ = ops.layer_norm_bwd(dy, x, stats, w, True, False, False)
    assert torch.equal(dx, dx_only)


def test_the_result_has_the_inputs_type_under_autocast():
    m = LayerNorm(40).to(DEV)
    for x in (torch.randn(9, 40, device=DEV), torch.randn(9, 40, device=DEV).bfloat16()):
        want = m(x)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m(x)
            y.float().square().sum().backward()
        assert y.dtype == want.dtype == x.dtype and torch.equal(y, want) and m.weight.grad.dtype == torch.float32
    with pytest.raises(BtsAmdError):
        m.bfloat16()(x)


def test_checkpointed_and_offloaded_passes():
    """A slice of a wider buffer through torch.utils.checkpoint, whose recomputed tensors take the saved ones' place."""
    from torch.utils.checkpoint import checkpoint
    x, w, b, dy = make(300, 96, torch.float32, 97, pad=7)
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))

    def block(x):
        return layer_norm(torch.relu(layer_norm(x, w, b)) * 2, w, b)
    want = torch.autograd.grad(block(x), (x, w, b), dy)
    for reentrant in (True, False):
        got = []
        for t in (x, w, b):
            t.grad = None
        block_out = checkpoint(block, x, use_reentrant=reentrant)
        block_out.backward(dy)
        got = [t.grad for t in (x, w, b)]
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_saved_tensors_that_come_back_elsewhere_are_refused():
    """A hook that moves what is saved to the host and leaves it there: refused, the kernel must not see host memory."""
    x, w, b, dy = make(40, 64, torch.float32, 101)
    for only in (x, w):
        x, w, b = (t.detach().requires_grad_(True) for t in (x, w, b))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu() if t.shape == only.shape else t, lambda t: t):
            y = layer_norm(x, w, b)
        with pytest.raises(BtsAmdError):
            torch.autograd.grad(y, (x, w, b), dy)
