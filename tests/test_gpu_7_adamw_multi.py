"""FusedAdamW with 8-bit states, clipping and bf16 parameters (bts_adamw_multi_*) against the definition in 64 bits.

8-bit states are compared exactly: the kernel forms the moments in 64 bits and what it starts from is exact, so its codes are the
definition's.  u = 2^-24.  An update is off by at most 12 u of itself (m to f32, v to f32 under a root, root, reciprocal bias root and
its product, eps' sum, quotient, step size and its product, clip coefficient), taken with the magnitudes that meet in m, and the sum with
the decayed parameter by 3 u of that; 32-bit states: m by 5 u (|b1 m| + |a1 g|) (three constants, two products), v by 8 u."""
import copy

import pytest
import torch

from bts_amd._lib import BtsAmdError
from bts_amd.optim import FusedAdamW
from tests import adamw_ref as R

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
BETAS = (0.9, 0.999)
SIZES = [1, 3, 255, 256, 257, 1000, 4095, 4096, 4097, 12345, 70001]


def flat64(t, p=None):
    """Elements in memory order (of p, or of t itself), 64 bits on the CPU."""
    t = t.detach()
    p = t if p is None else p
    return torch.as_strided(t, (t.numel(),), (1,), t.storage_offset()).double().cpu() if t.stride() == p.stride() else t.flatten().double().cpu()


def optimizer(ps, cut=None, **kw):
    groups = [{"params": ps[:cut], "weight_decay": 1e-2}]
    if cut is not None and ps[cut:]:
        groups.append({"params": ps[cut:], "weight_decay": 0.0})
    kw = {"lr": 1e-3, "betas": BETAS, "eps": 1e-4, **kw}
    return FusedAdamW(groups, **kw)


def check_step(opt, **step_kw):
    """One opt.step() against the definition, from the state it finds."""
    ps = [p for g in opt.param_groups for p in g["params"] if p.grad is not None]
    decay = {id(p): (g["weight_decay"], g["lr"], g["betas"], g["eps"]) for g in opt.param_groups for p in g["params"]}
    t = opt.device_steps()[0] + 1
    had = {id(p): mv for p, mv in zip([p for g in opt.param_groups for p in g["params"]], opt.moments())}
    before = [(flat64(p), flat64(p.grad), flat64(had[id(p)][0]), flat64(had[id(p)][1])) for p in ps]
    norm, c = R.clip_of([p.grad for p in ps], opt.max_grad_norm) if opt.max_grad_norm is not None else (None, 1.0)
    grads = [p.grad.clone() for p in ps]
    opt.step(**step_kw)
    now = {id(p): mv for p, mv in zip([p for g in opt.param_groups for p in g["params"]], opt.moments())}
    torch.cuda.synchronize()
    if norm is not None:
        assert abs(opt.grad_norm.item() - norm) <= 2 * U * norm
    for p, g0, (p0, g, m, v) in zip(ps, grads, before):
        wd, lr, betas, eps = decay[id(p)]
        p1, m1, v1, upd, mag = R.step(p0, g, m, v, t, lr, betas, eps, wd, c)
        what = (tuple(p.shape), p.dtype)
        assert torch.equal(p.grad, g0), what
        tol = 12 * U * upd + 3 * U * (p1.abs() + upd)
        if p.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * (p1.abs() + tol)
        off = (flat64(p) - p1).abs() - tol
        assert off.max().item() <= 0, (what, off.max().item(), off.argmax().item())
        got_m, got_v = (flat64(x) for x in now[id(p)])
        if "exp_avg_codes" in opt.state[p]:
            (want_m, km), (want_v, kv) = R.hold(m1, True), R.hold(v1, False)
            assert torch.equal(got_m, want_m), (what, (got_m != want_m).nonzero().flatten()[:5])
            assert torch.equal(got_v, want_v), (what, (got_v != want_v).nonzero().flatten()[:5])
            assert opt.state[p]["exp_avg_scales"].tolist() == [2.0 ** k for k in km]
            assert opt.state[p]["exp_avg_sq_scales"].tolist() == [2.0 ** k for k in kv]
        else:
            assert ((got_m - m1).abs() <= 5 * U * mag).all() and ((got_v - v1).abs() <= 8 * U * v1).all(), what


def tensors(sizes, dtype, seed, requires_grad=True):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(n, generator=gen, device=DEV).mul_(0.1).to(dtype).requires_grad_(requires_grad) for n in sizes]


def feed(ps, seed, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for i, p in enumerate(ps):
        g = torch.empty_like(p).copy_(torch.randn(p.shape, generator=gen, device=DEV) * scale * 10.0 ** -(i % 5))
        g.view(-1)[::7] = 0 if g.is_contiguous() else g.view(-1)[::7]
        if p.grad is None:
            p.grad = g
        else:
            p.grad.copy_(g)


@pytest.mark.parametrize("clip", [None, 0.5, float("inf")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits,least", [(8, 4096), (8, 1), (32, 4096)])
def test_steps_against_the_definition(bits, least, dtype, clip):
    ps = tensors(SIZES, dtype, 1)
    opt = optimizer(ps, 6, state_bits=bits, max_grad_norm=clip, min_8bit_size=least)
    for it in range(4):
        feed(ps, 10 + it)
        opt.param_groups[0]["lr"] = 1e-3 * (1 - it / 10)
        check_step(opt)
    assert [("exp_avg_codes" in opt.state[p]) for p in ps] == [bits == 8 and n >= least for n in SIZES]
    assert opt.device_steps() == [4.0, 4.0]


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-11])
@pytest.mark.parametrize("bits", [8, 32])
def test_small_eps_and_small_gradients(bits, eps):
    """An eps that keeps nothing away from zero: gradients of 1e-14 .. 1e-8 (their squares are still normal f32 numbers) and the other
    betas; lr 0 and no decay move nothing."""
    gen = torch.Generator(device=DEV).manual_seed(43)
    p = torch.randn(6000, generator=gen, device=DEV).requires_grad_(True)
    opt = FusedAdamW([p], lr=1e-2, betas=(0.0, 0.5), eps=eps, weight_decay=0.0, state_bits=bits)
    for it in range(3):
        g = torch.randn(6000, generator=gen, device=DEV)
        p.grad = torch.where(g.abs() < 1e-3, torch.full_like(g, 1e-3), g) * torch.logspace(-11, -8, 6000, device=DEV)
        check_step(opt)
    opt.param_groups[0]["lr"] = 0.0
    was = p.detach().clone()
    check_step(opt)
    assert torch.equal(p, was)


def test_without_options_the_step_stays_what_it_was():
    """f32 parameters and no option: bts_adamw_step, whose 1 - beta2 is formed in f32 (0.00100004673).  bf16 parameters move to the
    multi-tensor kernel by themselves."""
    p = tensors([5000], torch.float32, 41)[0]
    p.grad = torch.full_like(p, 2.0)
    opt = FusedAdamW([p])
    assert opt.state_bits == 32 and opt.max_grad_norm is None
    opt.step()
    assert (opt.state[p]["exp_avg_sq"] == (torch.tensor(1.0) - torch.tensor(0.999)).item() * 2.0 * 2.0).all()
    q = tensors([5000], torch.bfloat16, 41)[0]
    q.grad = torch.full_like(q, 2.0)
    opt = FusedAdamW([q])
    opt.step()
    assert ((opt.state[q]["exp_avg_sq"] - 0.004).abs() <= 4 * U * 0.004).all()


def test_mixed_types_in_one_step():
    ps = tensors([5000, 300], torch.float32, 2) + tensors([9000, 77], torch.bfloat16, 3)
    opt = optimizer(ps, 3, state_bits=8, max_grad_norm=0.1)
    for it in range(3):
        feed(ps, 20 + it)
        check_step(opt)


@pytest.mark.parametrize("signed", [True, False])
def test_every_code_and_its_border(signed):
    """All numbers of the form, at several scales, come back as they are; midpoints go to the even neighbour, their neighbours in f32 to
    the nearer one."""
    x = R.numbers(signed)
    mids = (x[1:] + x[:-1]) / 2
    up = torch.nextafter(mids.float(), torch.tensor(float("inf"))).double()
    down = torch.nextafter(mids.float(), torch.tensor(0.0)).double()
    rows = []
    for k in (0, -10, -126, 60, 100):
        for vals in (x, mids, up, down):
            blk = torch.zeros(256, dtype=torch.float64)
            blk[:vals.numel()] = vals
            if vals.numel() < 256:
                blk[255] = x[-1]                                            # holds the block's scale
            else:
                blk[0] = x[-1]
            if signed:
                blk[1:200:2] *= -1
            rows.append(blk * 2.0 ** k)
    blk = torch.cat(rows)
    blk = blk.float().double()                                              # what a checkpoint holds
    p = torch.zeros(blk.numel(), device=DEV, requires_grad=True)
    opt = FusedAdamW([p], state_bits=8, min_8bit_size=1)
    sd = opt.state_dict()
    other = torch.ones_like(p)
    mine = blk.float().to(DEV)
    sd["state"] = {0: {"step": torch.tensor(3.0), "exp_avg": mine if signed else other, "exp_avg_sq": other if signed else mine}}
    opt.load_state_dict(sd)
    got = opt.moments(flat=True)[0 if signed else 1].double().cpu()
    want, ks = R.hold(blk, signed)
    assert torch.equal(got, want)
    assert opt.state[p]["exp_avg_scales" if signed else "exp_avg_sq_scales"].tolist() == [2.0 ** k for k in ks]
    again = copy.deepcopy(opt.state_dict())                                 # values that came from codes give the same values
    opt.load_state_dict(again)
    assert torch.equal(opt.moments(flat=True)[0 if signed else 1].double().cpu(), want)
    assert opt.device_steps() == [3.0]


def test_blocks_with_extreme_values():
    """Zeros, one outlier, far apart magnitudes, the smallest and the largest f32 values."""
    gen = torch.Generator().manual_seed(5)
    rows = [torch.zeros(256), torch.full((256,), 1e-45), torch.full((256,), 3.4e38), torch.randn(256, generator=gen) * 1e-38, torch.randn(256, generator=gen) * 1e30,
            torch.randn(256, generator=gen) * 10.0 ** torch.linspace(-40, 30, 256), torch.linspace(-1, 1, 256) * 3.0, torch.randn(200, generator=gen)]
    rows[0][17] = 2.0
    x = torch.cat(rows)
    p = torch.zeros(x.numel(), device=DEV, requires_grad=True)
    opt = FusedAdamW([p], state_bits=8, min_8bit_size=1)
    sd = opt.state_dict()
    sd["state"] = {0: {"step": torch.tensor(1.0), "exp_avg": x, "exp_avg_sq": x.abs()}}
    opt.load_state_dict(sd)
    m, v = (t.double().cpu() for t in opt.moments(flat=True))
    want = R.hold(x.double(), True)[0]
    over = x == 3.4e38                                                      # 2^128 in four bits: beyond the form, like infinity
    assert over.sum() == 256 and torch.isnan(want[over]).all() and torch.isnan(m[over]).all()
    assert torch.equal(m[~over], want[~over])
    want = R.hold(x.abs().double(), False)[0]
    assert torch.equal(v, want) and ((v > 0) == (x != 0)).all()


def test_values_that_are_not_finite_keep_to_themselves():
    p = torch.zeros(1024, device=DEV, requires_grad=True)
    q = torch.zeros(1024, device=DEV, requires_grad=True)
    oa, ob = FusedAdamW([p], state_bits=8, min_8bit_size=1), FusedAdamW([q], state_bits=8, min_8bit_size=1)
    g = torch.randn(1024, device=DEV)
    bad = g.clone()
    bad[5], bad[300], bad[301] = float("nan"), float("inf"), -float("inf")
    for it in range(2):
        p.grad, q.grad = bad.clone(), g.clone()
        oa.step()
        ob.step()
    where = torch.zeros(1024, dtype=torch.bool, device=DEV)
    where[[5, 300, 301]] = True
    ma, va = oa.moments(flat=True)
    mb, vb = ob.moments(flat=True)
    # a block's scale is taken without them: where they were not its largest values, the others do not change at all
    assert torch.equal(p[~where], q[~where])
    assert torch.isnan(ma[where]).all() and torch.isnan(va[5]) and torch.isinf(va[[300, 301]]).all()
    assert torch.isfinite(ma[~where]).all() and torch.isfinite(va[~where]).all()
    big = torch.zeros(300, device=DEV, requires_grad=True)                   # g^2 beyond f32: v is infinite, the parameter does not move
    o = FusedAdamW([big], state_bits=8, min_8bit_size=1, weight_decay=0.0)
    big.grad = torch.full((300,), 1e30, device=DEV)
    o.step()
    assert (big == 0).all() and torch.isinf(o.moments(flat=True)[1]).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_only_the_tensors_change(bits):
    """Parameters and gradients are views at odd offsets of larger buffers; what lies around them stays."""
    sizes, gap = [4097, 300, 5003, 1], 3
    buf = {k: torch.full((sum(sizes) + gap * 5,), 7.0, device=DEV, dtype=d) for k, d in (("p", torch.float32), ("b", torch.bfloat16))}
    ps, mask = [], {k: torch.ones_like(t, dtype=torch.bool) for k, t in buf.items()}
    for k in buf:
        at = gap
        for n in sizes:
            p = torch.nn.Parameter(buf[k][at:at + n])
            p.data.copy_(torch.randn(n, device=DEV))
            mask[k][at:at + n] = False
            ps.append(p)
            at += n + gap
    opt = optimizer(ps, 4, state_bits=bits, max_grad_norm=1.0, min_8bit_size=256)
    for it in range(2):
        for p in ps:
            g = torch.randn(p.numel() + 5, device=DEV).to(p.dtype)
            p.grad = g[5:] if it else g[:-5]
        check_step(opt)
    for k in buf:
        assert (buf[k][mask[k]] == 7.0).all()


def test_channels_last_parameters_and_checkpoints_of_the_other_layout():
    torch.manual_seed(0)
    w = torch.randn(40, 24, 3, 3, device=DEV)
    a = w.clone().contiguous(memory_format=torch.channels_last).requires_grad_(True)
    b = w.clone().requires_grad_(True)
    for kw in (dict(state_bits=8, min_8bit_size=1), dict(max_grad_norm=1e9), dict()):
        oa, ob = FusedAdamW([a], eps=1e-3, **kw), torch.optim.AdamW([b], eps=1e-3)
        with torch.no_grad():
            a.copy_(w)
            b.copy_(w)
        g = torch.randn_like(w)
        a.grad, b.grad = g.clone().contiguous(memory_format=torch.channels_last), g.clone()
        oa.step()
        ob.step()
        assert (a - b).abs().max() <= 1e-6
        oa.load_state_dict(copy.deepcopy(ob.state_dict()))                  # contiguous moments for a channels-last parameter
        sa = oa.state_dict()["state"][0]
        assert sa["exp_avg"].stride() == a.stride() and sa["exp_avg"].shape == a.shape
        ref = ob.state_dict()["state"][0]["exp_avg"]
        err = (sa["exp_avg"] - ref).abs()
        assert (err <= 2.0 ** -4 * ref.abs() + 2.0 ** -18 * ref.abs().max()).all() if "state_bits" in kw else torch.equal(sa["exp_avg"], ref)
        oa.step()
        ob.step()
        assert (a - b).abs().max() <= (3e-4 if "state_bits" in kw else 1e-6)     # an update is at most lr = 1e-3, its relative error 2^-4 + 2^-5
    with pytest.raises(BtsAmdError):
        o = FusedAdamW([a], state_bits=8)
        a.grad = g.clone()                                                  # the gradient's order is not the parameter's
        o.step()


def test_gradients_that_come_and_go():
    ps = tensors([5000, 40, 7000], torch.float32, 7)
    opt = optimizer(ps, 2, state_bits=8, max_grad_norm=1.0)
    assert opt.grad_norm is None
    opt.step()                                                              # no gradient at all: only the step count moves
    assert opt.device_steps() == [1.0, 1.0] and not opt.state and opt.grad_norm.item() == 0.0
    feed(ps[:2], 1)
    check_step(opt)
    feed(ps, 2)
    check_step(opt)
    keep = []
    for it in range(3):                                                     # new gradient tensors every step
        opt.zero_grad(set_to_none=True)
        keep.append(torch.empty(1000 + it, device=DEV))
        feed(ps[it % 2:], 3 + it)
        check_step(opt)
    assert opt.device_steps() == [6.0, 6.0]


def test_checkpoints_are_torch_ones():
    """torch.optim.AdamW's state loads into 8 bits (each value to its nearest code) and the other way round (exactly)."""
    torch.manual_seed(0)
    ws = [torch.randn(70, 80, device=DEV), torch.randn(9, device=DEV)]
    a, b = [w.clone().requires_grad_(True) for w in ws], [w.clone().requires_grad_(True) for w in ws]
    ob = torch.optim.AdamW(b, lr=1e-3, eps=1e-3)
    for it in range(5):
        for q in b:
            q.grad = torch.randn_like(q)
        ob.step()
    oa = FusedAdamW(a, lr=1e-3, eps=1e-3, state_bits=8, min_8bit_size=100)
    oa.load_state_dict(copy.deepcopy(ob.state_dict()))
    assert oa.device_steps() == [5.0] and oa.param_groups[0]["eps"] == 1e-3
    for i, p in enumerate(a):
        m, v = oa.moments()[i]
        sb = ob.state_dict()["state"][i]
        if i == 0:
            assert torch.equal(flat64(m), R.hold(flat64(sb["exp_avg"]), True)[0]) and torch.equal(flat64(v), R.hold(flat64(sb["exp_avg_sq"]), False)[0])
        else:
            assert torch.equal(m, sb["exp_avg"]) and torch.equal(v, sb["exp_avg_sq"])
    sa = oa.state_dict()
    assert all(set(s) == {"step", "exp_avg", "exp_avg_sq"} and float(s["step"]) == 5.0 for s in sa["state"].values())
    ob.load_state_dict(copy.deepcopy(sa))
    for i in range(2):
        assert torch.equal(ob.state_dict()["state"][i]["exp_avg"], oa.moments()[i][0])
    for p in a:
        p.grad = torch.randn_like(p)
    check_step(oa)


def test_bf16_parameters_keep_f32_moments_through_a_checkpoint():
    ps = tensors([5000, 64], torch.bfloat16, 11)
    opt = optimizer(ps, 1, max_grad_norm=1.0)
    feed(ps, 1)
    check_step(opt)
    sd = copy.deepcopy(opt.state_dict())
    assert sd["state"][0]["exp_avg"].dtype == torch.float32
    other = optimizer(ps, 1, max_grad_norm=1.0)
    other.load_state_dict(sd)
    assert all(torch.equal(x, y) for x, y in zip(opt.moments(flat=True), other.moments(flat=True)))
    check_step(other)


def test_clipped_f32_step_is_torchs():
    torch.manual_seed(3)
    ws = [torch.randn(64, 33, device=DEV), torch.randn(7, device=DEV)]
    a, b = [w.clone().requires_grad_(True) for w in ws], [w.clone().requires_grad_(True) for w in ws]
    oa, ob = FusedAdamW(a, lr=1e-3, eps=1e-3, max_grad_norm=0.7), torch.optim.AdamW(b, lr=1e-3, eps=1e-3)
    for it in range(3):
        for p, q in zip(a, b):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
        norm = torch.nn.utils.clip_grad_norm_(b, 0.7)
        oa.step()
        ob.step()
        assert abs(oa.grad_norm - norm) <= 1e-6 * norm
        assert all((p - q).abs().max() <= 1e-6 for p, q in zip(a, b))


def test_norm_of_large_small_and_broken_gradients():
    ps = tensors([3000, 5], torch.float32, 13)
    opt = optimizer(ps, None, max_grad_norm=1.0)
    for value in (1e25, 1e-25):
        for p in ps:
            p.grad = torch.full_like(p, value)
        opt.step()
        assert abs(opt.grad_norm.item() / value - 3005 ** 0.5) <= 1e-5 and all(torch.isfinite(p).all() for p in ps)
    ps[1].grad[2] = float("nan")
    opt.step()                                                              # torch's rule: the coefficient is NaN, so is everything
    assert torch.isnan(opt.grad_norm) and all(torch.isnan(p).all() for p in ps)


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_replay(bits):
    ps, qs = tensors([9000, 333], torch.float32, 17), tensors([9000, 333], torch.float32, 17)
    oa, ob = optimizer(ps, 1, state_bits=bits, max_grad_norm=0.5), optimizer(qs, 1, state_bits=bits, max_grad_norm=0.5)

    def eager(it):
        feed(qs, 30 + it)
        for g in ob.param_groups:
            g["lr"] = 1e-3 / (it + 1)
        ob.step()
    with pytest.raises(BtsAmdError):                                        # no tables yet: refused, not recorded wrongly
        feed(ps, 30)
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            oa.step(prepared=True)
    torch.cuda.synchronize()
    feed(ps, 30)
    oa.prepare_step()
    oa.step(prepared=True)
    eager(0)
    with pytest.raises(BtsAmdError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            oa.moments()
    torch.cuda.synchronize()
    oa.moments()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        oa.step(prepared=True)
    with torch.cuda.graph(g2):
        oa.step(prepared=True)
        out = oa.moments(flat=True)
    for it in range(1, 6):
        feed(ps, 30 + it)
        oa.prepare_step([1e-3 / (it + 1)] * 2)
        (g1 if it % 2 else g2).replay()
        eager(it)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), it
        assert torch.equal(oa.grad_norm, ob.grad_norm)
        if it % 2 == 0:
            assert all(torch.equal(x, y) for x, y in zip(out, ob.moments(flat=True)))
    assert oa.device_steps() == [6.0, 6.0]
    # the graphs' tables stay theirs after the optimizer has made new ones
    for p in ps:
        p.grad = None
    feed(ps, 99)
    feed(qs, 99)
    for ga, gb in zip(oa.param_groups, ob.param_groups):                    # the replays took theirs from prepare_step's argument
        ga["lr"] = gb["lr"]
    oa.step()
    ob.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_a_graph_outlives_what_it_was_captured_with():
    """After the gradients are gone and a checkpoint is loaded, a replay still writes its own states and nothing else."""
    ps = tensors([9000, 333], torch.float32, 37)
    opt = optimizer(ps, 1, state_bits=8, max_grad_norm=0.5)
    feed(ps, 1)
    opt.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step(prepared=True)
    sd = copy.deepcopy(opt.state_dict())
    opt.zero_grad(set_to_none=True)
    opt.load_state_dict(sd)
    fence = [torch.full((9000,), 3.0, device=DEV) for _ in range(64)]       # takes what the allocator has free
    before = [t.clone() for t in opt.moments(flat=True)]
    g.replay()
    torch.cuda.synchronize()
    assert all((t == 3.0).all() for t in fence)
    assert all(torch.equal(a, b) for a, b in zip(before, opt.moments(flat=True))) and opt.device_steps() == [1.0, 1.0]


def test_steps_on_several_streams():
    ps, qs = tensors([50000, 333], torch.float32, 19), tensors([50000, 333], torch.float32, 19)
    oa, ob = optimizer(ps, 1, state_bits=8, max_grad_norm=0.5), optimizer(qs, 1, state_bits=8, max_grad_norm=0.5)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for it in range(6):
        s = streams[it % 2]
        s.wait_stream(torch.cuda.current_stream())
        s.wait_stream(streams[1 - it % 2])
        with torch.cuda.stream(s):
            for p in ps:
                p.grad = None
            feed(ps, 50 + it)
            oa.step()
        feed(qs, 50 + it)
        ob.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_groups_added_later():
    ps = tensors([5000, 300], torch.float32, 23)
    for kw in (dict(state_bits=8), dict()):
        opt = optimizer(ps[:1], None, **kw)
        feed(ps, 1)
        opt.step()
        opt.add_param_group({"params": ps[1:], "weight_decay": 0.0})
        opt.step()
        assert opt.device_steps() == [2.0, 1.0]
    opt.add_param_group({"params": tensors([600], torch.bfloat16, 3)})       # bf16 joins: from here on the multi-tensor kernels
    feed([p for g in opt.param_groups for p in g["params"]], 2)
    opt.step()
    assert opt.device_steps() == [3.0, 2.0, 1.0]


@pytest.mark.parametrize("kw", [dict(state_bits=8, min_8bit_size=1), dict(state_bits=8, max_grad_norm=1.0), dict()])
def test_copies_go_on_by_themselves(kw):
    """copy.deepcopy of a model with its optimizer: the copy has the states and the step count, and memory of its own."""
    ps = tensors([5001, 40], torch.float32, 31)
    opt = optimizer(ps, 1, **kw)
    feed(ps, 1)
    opt.step()
    qs, twin = copy.deepcopy((ps, opt))
    assert twin.device_steps() == [1.0, 1.0] and twin.param_groups[0]["params"][0] is qs[0]
    was = [p.detach().clone() for p in ps]
    feed(qs, 2)
    twin.step()
    assert all(torch.equal(p, w) for p, w in zip(ps, was))
    feed(ps, 2)
    opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and not torch.equal(ps[0], was[0])


def test_offsets_beyond_32_bits():
    """A bf16 parameter of 2^31 + 4613 elements: its last blocks are updated like those of a short tensor."""
    n, tail = 2 ** 31 + 4613, 5000
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of free device memory")
    p, q = torch.zeros(n, dtype=torch.bfloat16, device=DEV, requires_grad=True), None
    first = (n - tail) // 256 * 256
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g[first:] = torch.randn(n - first, device=DEV).to(torch.bfloat16)
    p.grad = g
    q = torch.zeros(n - first, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    q.grad = g[first:].clone()
    oa, ob = (optimizer([t], None, state_bits=8, min_8bit_size=1, max_grad_norm=1.0) for t in (p, q))
    oa.step()
    ob.step()
    assert torch.equal(p[first:], q) and (p[first - 4096:first] == 0).all() and oa.grad_norm == ob.grad_norm
    assert torch.equal(oa.state[p]["exp_avg_codes"][first:], ob.state[q]["exp_avg_codes"])
    assert torch.equal(oa.state[p]["exp_avg_sq_scales"][first // 256:], ob.state[q]["exp_avg_sq_scales"])


def test_refusals_on_the_device():
    a, b = tensors([5000, 5000], torch.float32, 29)
    for bad in (lambda: FusedAdamW([a.detach().half().requires_grad_(True)], state_bits=8), lambda: FusedAdamW([a.detach().double().requires_grad_(True)], max_grad_norm=1.0)):
        o = bad()
        o.param_groups[0]["params"][0].grad = torch.ones_like(o.param_groups[0]["params"][0])
        with pytest.raises(BtsAmdError):
            o.step()
    buf = torch.zeros(9000, device=DEV)
    overlap = [torch.nn.Parameter(buf[:5000]), torch.nn.Parameter(buf[4000:])]
    holes = [torch.nn.Parameter(buf[::2])]
    for ps in (overlap, holes):
        o = FusedAdamW(ps, state_bits=8)
        for p in ps:
            p.grad = torch.ones_like(p)
        with pytest.raises(BtsAmdError):
            o.step()
        assert (buf == 0).all()
    o = FusedAdamW([a, b], state_bits=8)
    sd = o.state_dict()
    sd["state"] = {0: {"step": torch.tensor(1.0), "exp_avg": torch.zeros(3), "exp_avg_sq": torch.zeros(5000)}}
    with pytest.raises(BtsAmdError):
        o.load_state_dict(sd)
    with pytest.raises(BtsAmdError):
        o.step(closure=lambda: None)


def test_normalised_head_trained_with_clipped_8bit_steps():
    """The operators together, as a training step uses them: LayerNorm2d -> 1x1 convolution -> loss, backward, clipped step with 8-bit
    states.  Every gradient against 64-bit autograd at the same parameters, every update against the definition from that gradient."""
    from bts_amd.norm import LayerNorm2d
    torch.manual_seed(0)
    norm, conv = LayerNorm2d(32).to(DEV), torch.nn.Conv2d(32, 160, 1, bias=False).to(DEV)
    net = torch.nn.Sequential(norm, conv)
    x = torch.randn(2, 32, 24, 20, device=DEV).contiguous(memory_format=torch.channels_last)
    target = torch.randn(2, 160, 24, 20, device=DEV)
    opt = FusedAdamW([{"params": norm.parameters(), "weight_decay": 0.0}, {"params": conv.parameters(), "weight_decay": 1e-2}], lr=1e-2, eps=1e-4,
                     state_bits=8, max_grad_norm=0.05)
    assert [p.numel() for p in net.parameters()] == [32, 32, 5120]
    for it in range(4):
        opt.zero_grad(set_to_none=it % 2 == 0)
        loss = (net(x) - target).square().mean()
        loss.backward()
        ref = [p.detach().double().cpu().requires_grad_(True) for p in net.parameters()]
        xr = x.double().cpu()
        mu, var = xr.mean(1, keepdim=True), xr.var(1, keepdim=True, correction=0)
        h = (xr - mu) / (var + 1e-5).sqrt() * ref[0].view(1, -1, 1, 1) + ref[1].view(1, -1, 1, 1)
        y = torch.nn.functional.conv2d(h, ref[2])
        (y - target.double().cpu()).square().mean().backward()
        for p, r in zip(net.parameters(), ref):
            # sums of 960 x 160 products of O(1) terms in f32, each with a few roundings: 2^-24 x 200 of the largest gradient
            assert (p.grad.double().cpu() - r.grad).abs().max() <= 200 * U * r.grad.abs().max() + 1e-9
        check_step(opt)
    assert "exp_avg_codes" in opt.state[conv.weight] and "exp_avg" in opt.state[norm.weight]


@pytest.mark.parametrize("bits", [8, 32])
def test_a_parameter_that_shrinks_in_place_is_refused(bits):
    p = tensors([9000], torch.float32, 47)[0]
    opt = optimizer([p], None, state_bits=bits)
    feed([p], 1)
    check_step(opt)
    whole = p.detach()
    was = whole.clone()
    p.data = p.data[:5000]
    p.grad = torch.ones(5000, device=DEV)
    for use in (opt.step, opt.moments, opt.state_dict):
        with pytest.raises(BtsAmdError):
            use()
    assert torch.equal(whole, was)
    p.data = whole
    p.grad = None
    feed([p], 2)
    check_step(opt)


def test_memory_dropped_while_another_stream_steps():
    """Tables, rows and states that were made on one stream and are dropped there while a step on another one still has to run: nobody else
    gets them before."""
    ps, qs = tensors([9000, 333], torch.float32, 59), tensors([9000, 333], torch.float32, 59)
    oa, ob = optimizer(ps, 1, state_bits=8, max_grad_norm=0.5), optimizer(qs, 1, state_bits=8, max_grad_norm=0.5)
    for o, ts in ((oa, ps), (ob, qs)):
        feed(ts, 1)
        o.step()
    sd = copy.deepcopy(oa.state_dict())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for p in ps:
            p.grad = None
        feed(ps, 2)                                                         # other gradients: new records on this stream, the chunks stay
        torch.cuda._sleep(100000000)
        oa.step()
    oa.load_state_dict(sd)                                                  # drops the table, the rows and the states
    fence = [torch.full((n,), 3.0, device=DEV) for n in (4, 40, 300, 1000, 9000) * 40]
    torch.cuda.synchronize()
    assert all((t == 3.0).all() for t in fence)
    feed(qs, 2)
    ob.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and oa.device_steps() == [1.0, 1.0]


@pytest.mark.parametrize("bits", [8, 32])
def test_a_parameter_that_changes_its_order_in_memory(bits):
    """channels_last between two steps: refused until the state is loaded again, and then right."""
    torch.manual_seed(71)
    p = torch.randn(40, 24, 3, 3, device=DEV).requires_grad_(True)
    opt = optimizer([p], None, state_bits=bits)
    feed([p], 1)
    check_step(opt)
    m, v = (t.clone() for t in opt.moments()[0])
    p.data = p.data.contiguous(memory_format=torch.channels_last)
    p.grad = torch.randn_like(p)
    was = p.detach().clone()
    with pytest.raises(BtsAmdError):
        opt.step()
    assert torch.equal(p, was) and all(torch.equal(a, b) for a, b in zip(opt.moments()[0], (m, v)))
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    m1, v1 = opt.moments()[0]
    assert m1.stride() == p.stride()
    if bits == 32:
        assert torch.equal(m1, m) and torch.equal(v1, v)
    else:                                                                   # other 256 elements share a scale now
        assert ((m1 - m).abs() <= 2.0 ** -4 * m.abs() + 2.0 ** -18 * m.abs().max()).all() and ((v1 - v).abs() <= 2.0 ** -4 * v + 2.0 ** -30 * v.max()).all()
    check_step(opt)


def test_a_graph_outlives_the_memory_of_its_parameters():
    """Parameter and gradient are given other memory after the capture: a replay writes what it was captured with, and nothing else."""
    ps = tensors([9000, 333], torch.float32, 73)
    opt = optimizer(ps, 1, state_bits=8, max_grad_norm=0.5)
    feed(ps, 1)
    opt.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step(prepared=True)
    for p in ps:
        p.data = p.data.clone()
        p.grad = None
    torch.cuda.synchronize()
    now = [p.detach().clone() for p in ps]
    fence = [torch.full((n,), 3.0, device=DEV) for n in (9000, 333) * 64]   # takes what the allocator has free
    g.replay()
    torch.cuda.synchronize()
    assert all((t == 3.0).all() for t in fence) and all(torch.equal(p, n) for p, n in zip(ps, now))


@pytest.mark.parametrize("kw", [dict(state_bits=8), dict(max_grad_norm=1.0), dict()])
def test_state_dict_hooks_see_and_change_the_moments(kw):
    """torch's contract: a post hook of state_dict sees what is returned, what a pre hook of load_state_dict returns is loaded, and its post
    hook finds the state in place."""
    ps = tensors([5000, 40], torch.float32, 79)
    opt = optimizer(ps, 1, **kw)
    feed(ps, 1)
    opt.step()
    seen = []

    def after(o, sd):
        seen.append({i: st["exp_avg"].clone() for i, st in sd["state"].items()})
        for i, st in sd["state"].items():                                   # (without options these dicts are the optimizer's own: not in place)
            sd["state"][i] = {**st, "exp_avg": st["exp_avg"] * 2.0}
    handles = [opt.register_state_dict_post_hook(after)]
    sd = opt.state_dict()
    handles[0].remove()
    plain_sd = copy.deepcopy(opt.state_dict())
    for i in (0, 1):
        assert torch.equal(seen[0][i], plain_sd["state"][i]["exp_avg"]) and torch.equal(sd["state"][i]["exp_avg"], 2.0 * seen[0][i])

    def before(o, sd):
        sd = copy.deepcopy(sd)
        for st in sd["state"].values():
            st["exp_avg"] = st["exp_avg"] * 4.0
            st["step"] = torch.tensor(9.0)
        return sd
    found = []
    handles = [opt.register_load_state_dict_pre_hook(before), opt.register_load_state_dict_post_hook(lambda o: found.append((o.state_dict(), o.device_steps())))]
    opt.load_state_dict(plain_sd)
    for h in handles:
        h.remove()
    now = opt.state_dict()
    assert opt.device_steps() == found[0][1] == [9.0, 9.0] and plain_sd["state"][0]["step"] == 1.0
    for i in (0, 1):                                                        # times a power of two: exact in 8 bits
        assert torch.equal(now["state"][i]["exp_avg"], 4.0 * plain_sd["state"][i]["exp_avg"]) and torch.equal(found[0][0]["state"][i]["exp_avg"], now["state"][i]["exp_avg"])
    assert not opt._optimizer_load_state_dict_pre_hooks and not opt._optimizer_load_state_dict_post_hooks and not opt._optimizer_state_dict_post_hooks


@pytest.mark.parametrize("bits", [8, 32])
def test_states_that_were_reset_begin_at_zero(bits):
    from collections import defaultdict
    ps = tensors([5000, 333], torch.float32, 83)
    opt = optimizer(ps, 1, state_bits=bits)
    for reset in (lambda: None, lambda: setattr(opt, "state", defaultdict(dict)), lambda: opt.state.update({ps[0]: {}}), lambda: opt.state.clear()):
        feed(ps, 1)
        check_step(opt)
        reset()
    assert all((t == 0).all() for mv in opt.moments() for t in mv)
    check_step(opt)


@pytest.mark.parametrize("bits", [8, 32])
def test_an_infinite_bound_only_measures(bits):
    """Also where the norm is infinite or NaN: the step is the one without a bound."""
    for bad in (float("inf"), float("nan"), -float("inf")):
        ps, qs = tensors([5000, 333], torch.float32, 89), tensors([5000, 333], torch.float32, 89)
        oa, ob = optimizer(ps, 1, state_bits=bits, max_grad_norm=float("inf")), optimizer(qs, 1, state_bits=bits)
        feed(ps, 1)
        feed(qs, 1)
        ps[0].grad[17] = qs[0].grad[17] = bad
        oa.step()
        ob.step()
        assert not torch.isfinite(oa.grad_norm) and torch.isnan(oa.grad_norm) == (bad != bad)
        for p, q in zip(ps, qs):
            assert torch.equal(torch.nan_to_num(p), torch.nan_to_num(q)) and torch.isnan(p).sum() == torch.isnan(q).sum() <= 1
        assert torch.isfinite(ps[1]).all()
