"""Host side of the layer normalisation: layouts, refusals of the wrappers and of the C entries (no GPU needed: every refused call
returns before a launch)."""
import ctypes as C

import pytest
import torch

from bts_amd import _lib, ops
from bts_amd.norm import LayerNorm, LayerNorm2d, layer_norm


def test_row_stride():
    t = torch.empty(4, 5, 6)
    assert ops.row_stride(t) == (20, 6)
    assert ops.row_stride(t[:, :, 1:4]) == (20, 6)
    assert ops.row_stride(t[:, 1:3]) is None                       # rows in groups
    assert ops.row_stride(t[1:2, 1:3]) == (2, 6)
    assert ops.row_stride(t.transpose(1, 2)) is None               # last axis not contiguous
    assert ops.row_stride(t[0, 0]) == (1, 6)
    assert ops.row_stride(t[..., :1]) == (20, 6)
    assert ops.row_stride(t[::2, :1]) == (2, 60)
    assert ops.row_stride(torch.empty(1, 6).expand(5, 6)) == (5, 0)
    assert ops.row_stride(torch.empty(1, 3, 6).expand(5, 3, 6)) is None
    assert ops.row_stride(torch.empty(0, 6)) == (0, 6)
    assert ops.row_stride(torch.empty(())) is None
    assert ops.row_stride(torch.empty(2, 8, 3, 5).contiguous(memory_format=torch.channels_last).permute(0, 2, 3, 1)) == (30, 8)


def test_cpu_tensors_are_refused():
    x = torch.randn(3, 8)
    for call in (lambda: layer_norm(x), lambda: LayerNorm(8)(x), lambda: LayerNorm2d(8)(torch.randn(1, 8, 2, 2)), lambda: ops.layer_norm_fwd(x)):
        with pytest.raises(_lib.BtsAmdError):
            call()


def test_c_entries_refuse_bad_arguments():
    lib, p, n = _lib.load(), C.c_void_p(4096), C.c_void_p(0)        # 4096: never read, the calls below end before any launch
    good = dict(x=p, dtype=0, xs=8, y=C.c_void_p(8192), ys=8, M=4, C=8, w=n, b=n, eps=1e-5, mean=n, rstd=n, st=n)
    fwd = lambda **k: lib.bts_layernorm_fwd(*{**good, **k}.values())   # noqa: E731
    for bad in (dict(x=n), dict(y=n), dict(y=p), dict(dtype=2), dict(dtype=-1), dict(M=0), dict(M=-3), dict(C=0), dict(xs=-1), dict(ys=7), dict(eps=-1.0),
                dict(eps=float("nan")), dict(mean=p), dict(rstd=p), dict(x=C.c_void_p(4098)), dict(y=C.c_void_p(8193), dtype=1)):
        assert fwd(**bad) == -1, bad
    assert fwd(C=16385, xs=16385, ys=16385) == -3
    good_b = dict(dy=p, dys=8, x=C.c_void_p(8192), xs=8, dx=C.c_void_p(16384), dxs=8, dtype=0, M=4, C=8, w=n, mean=p, rstd=p, dw=p, db=p, ws=p, st=n)
    bwd = lambda **k: lib.bts_layernorm_bwd(*{**good_b, **k}.values())   # noqa: E731
    for bad in (dict(dy=n), dict(x=n), dict(mean=n), dict(rstd=n), dict(ws=n), dict(ws=C.c_void_p(4097)), dict(dx=p), dict(dx=C.c_void_p(8192)), dict(dxs=7),
                dict(dtype=3), dict(M=0), dict(C=0), dict(dys=-8), dict(dx=n, dw=n, db=n)):
        assert bwd(**bad) == -1, bad
    assert bwd(C=16385, xs=16385, dys=16385, dxs=16385) == -3
    size = lib.bts_layernorm_bwd_workspace_bytes
    assert size(0, 10, 16385) == size(0, 0, 8) == size(2, 10, 8) == 0
    assert size(0, 1, 8) == 64 and size(1, 10 ** 9, 96) >= size(1, 10, 96) > 0


def test_modules_have_torch_parameters():
    assert [(k, tuple(v.shape)) for k, v in LayerNorm(12).state_dict().items()] == [(k, tuple(v.shape)) for k, v in torch.nn.LayerNorm(12).state_dict().items()]
    assert list(LayerNorm2d(12, bias=False).state_dict()) == ["weight"] and list(LayerNorm2d(12, elementwise_affine=False).state_dict()) == []


def test_adamw_options_are_checked():
    from bts_amd.optim import FusedAdamW
    p = torch.nn.Parameter(torch.zeros(8))
    for bad in (dict(state_bits=4), dict(state_bits=16), dict(state_bits=0), dict(max_grad_norm=0.0), dict(max_grad_norm=-1.0), dict(max_grad_norm=float("nan")),
                dict(min_8bit_size=0), dict(min_8bit_size=1.5)):
        with pytest.raises(_lib.BtsAmdError):
            FusedAdamW([p], **bad)
    o = FusedAdamW([p], state_bits=8)
    with pytest.raises(AttributeError):              # options are fixed: states and rows are laid out by them
        o.max_grad_norm = 1.0
    p.grad = torch.ones(8)
    with pytest.raises(_lib.BtsAmdError):            # no CPU path
        o.step()


def test_adamw_c_entries_refuse_bad_arguments():
    lib, p, n = _lib.load(), C.c_void_p(4096), C.c_void_p(0)
    hyper = (C.c_double * 6)()
    good = dict(t=p, c=p, nc=1, rows=p, ng=1, h=hyper, ws=p, gn=p, st=n)
    step = lambda **k: lib.bts_adamw_multi_step(*{**good, **k}.values())   # noqa: E731
    for bad in (dict(t=n), dict(c=n), dict(nc=0), dict(nc=-1), dict(nc=2 ** 24), dict(rows=n), dict(ng=0), dict(ng=65), dict(ws=n), dict(gn=n),
                dict(ws=C.c_void_p(4100))):
        assert step(**bad) == -1, bad
    assert lib.bts_adamw_multi_set(n, 1, hyper, n) == lib.bts_adamw_multi_set(p, 0, hyper, n) == lib.bts_adamw_multi_set(p, 1, n, n) == -1
    good_m = dict(t=p, c=p, nc=1, off=p, m=p, v=p, store=0, st=n)
    moments = lambda **k: lib.bts_adamw_multi_moments(*{**good_m, **k}.values())   # noqa: E731
    for bad in (dict(t=n), dict(c=n), dict(nc=0), dict(off=n), dict(m=n), dict(v=n), dict(store=2)):
        assert moments(**bad) == -1, bad
    assert lib.bts_adamw_multi_workspace_bytes() > 0


def test_adamw_record_matches_the_header():
    from bts_amd import optim
    src = open(_lib.os.path.join(_lib.os.path.dirname(_lib._HERE), "include", "bts_amd.h")).read()
    for name, value in (("CHUNK", optim._CHUNK), ("BLOCK", optim._BLOCK), ("ROW", optim._WIDE_ROW), ("MAX_GROUPS", optim._MAX_GROUPS)):
        assert "#define BTS_ADAMW_%s %d\n" % (name, value) in src
    assert optim._RECORD.itemsize == 64 and [optim._RECORD.fields[f][1] for f in ("p", "g", "m", "v", "m_scale", "v_scale", "n", "group", "flags")] == [
        0, 8, 16, 24, 32, 40, 48, 56, 60]


def test_the_written_down_8bit_forms():
    """The tests' own definition: spacing, range and rounding of the two forms."""
    from tests import adamw_ref as R
    s, u = R.numbers(True), R.numbers(False)
    assert s.numel() == 127 and s[-1] == 448 and s[1] == 2.0 ** -9 and u.numel() == 248 and u[-1] == 61440 and u[1] == 2.0 ** -17
    assert torch.equal(s, torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double())
    assert torch.equal(u, (torch.arange(248, dtype=torch.int32) << 7).to(torch.int16).view(torch.float16).double())
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(1000, generator=gen, dtype=torch.float64) * 10 ** torch.randn(1000, generator=gen, dtype=torch.float64)
    for signed in (True, False):
        a = x if signed else x.abs()
        y, ks = R.hold(a, signed)
        for b, k in zip(range(0, 1000, 256), ks):
            blk, got = a[b:b + 256], y[b:b + 256]
            assert ((got - blk).abs() <= 2.0 ** -4 * blk.abs() + 2.0 ** (k - (10 if signed else 18))).all()
            top = 448.0 if signed else 61440.0
            assert got.abs().max() <= top * 2.0 ** k and got.abs().max() > top * 2.0 ** (k - 1) * 0.96
        assert torch.equal(R.hold(y, signed)[0], y)


def test_every_width_has_a_kernel():
    """The rule for lanes and vectors (restated) covers every width of both types with a variant that the launcher lists, and of a row's
    vectors per lane only the last may be missing: the kernels load the others without a check."""
    src = open(_lib.os.path.join(_lib._HERE, "csrc", "layernorm.hip")).read()
    import re
    short = set(re.findall(r"LN_CASE\(T, (\d+), (\d+), F\)", src))
    have = {t: {(int(a), int(b)) for a, b in short | set(re.findall(r"LN_CASE\(%s, (\d+), (\d+), F\)" % t, src))} for t in ("F32", "BF16")}
    for t, vec in (("F32", 4), ("BF16", 8)):
        seen = set()
        for c in range(1, ops.LN_MAX_C + 1):
            nv = -(-c // vec)
            most = 1 if nv <= 64 else (16 if c <= 1024 or c > 8192 else 8) // vec
            lanes = 1
            while lanes * most < nv:
                lanes *= 2
            if nv > 64:
                lanes = 64 if c <= 1024 else -(-nv // 64) * 64 if vec == 8 and nv <= 384 else max(lanes, 256)
            k = -(-nv // lanes)
            assert (lanes, k) in have[t] and lanes * k >= nv > lanes * (k - 1), (t, c, lanes, k)
            seen.add((lanes, k))
        assert seen == have[t]                       # and every listed variant is some width's


@pytest.fixture
def stubbed_norm(monkeypatch):
    """layer_norm on CPU tensors: the launches are recorded, nothing is computed.  -> list of (name, x, its rows and stride) per launch."""
    seen = []

    def fwd(x, rows, weight, bias, eps, want_stats):
        seen.append(("fwd", x, rows))
        y = torch.zeros(x.shape, dtype=x.dtype)
        return (y, torch.zeros(2, rows[0])) if want_stats else y

    def bwd(dy, dys, x, rows, stats, weight, want_dx, want_dweight, want_dbias):
        seen.append(("bwd", x, rows))
        assert x.stride()[-1] == 1 and ops.row_stride(x) == rows and ops.row_stride(dy)[1] == dys and stats.shape == (2, rows[0])
        return tuple(torch.zeros(s, dtype=t) if w else None for w, s, t in zip(
            (want_dx, want_dweight, want_dbias), (x.shape, x.shape[-1:], x.shape[-1:]), (x.dtype, torch.float32, torch.float32)))
    monkeypatch.setattr(ops, "layer_norm_fwd_rows", fwd)
    monkeypatch.setattr(ops, "layer_norm_bwd_unchecked", bwd)
    monkeypatch.setattr(_lib, "require_gpu", lambda t: None)
    monkeypatch.setattr(ops, "current_device", lambda: -1)
    return seen


def test_backward_goes_by_the_layout_of_what_hooks_give_back(stubbed_norm):
    """A saved-tensor hook may give a strided input back dense: the launch must not walk it with the stride of the tensor that was saved
    (for 401 rows of 667 in 672 columns it would end 2000 elements behind it)."""
    w, b = torch.ones(667, requires_grad=True), torch.zeros(667, requires_grad=True)
    x = torch.randn(401, 672)[:, :667].requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t):
        layer_norm(x, w, b).sum().backward()
    assert stubbed_norm[-1][2] == (401, 672)
    for pack in (torch.clone, lambda t: t.contiguous().clone()):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            layer_norm(x, w, b).sum().backward()
        assert stubbed_norm[-1][0] == "bwd" and stubbed_norm[-1][1].shape == (401, 667) and stubbed_norm[-1][2] == (401, 667)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t()):     # another order in memory
        layer_norm(x, w, b).sum().backward()
    assert stubbed_norm[-1][2] == (401, 667)


@pytest.mark.parametrize("change", [lambda t: t.bfloat16(), lambda t: t[..., :-1], lambda t: t.double()])
def test_backward_refuses_other_values_than_were_saved(stubbed_norm, change):
    x = torch.randn(8, 16, requires_grad=True)
    for w, dtype in ((None, torch.float32), (torch.ones(16, requires_grad=True), torch.bfloat16)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            y = layer_norm(x.to(dtype), w)
        n = len(stubbed_norm)
        with pytest.raises(_lib.BtsAmdError):
            y.sum().backward()
        assert len(stubbed_norm) == n


@pytest.fixture
def stubbed_adamw(monkeypatch):
    """FusedAdamW with options on CPU tensors: no launch happens, each is recorded as (name, records of its table, chunks of its table)."""
    from bts_amd import optim
    launches, empty, tables = [], torch.empty, {}

    def table(self, *a):
        init(self, *a)
        tables[self.chunks.data_ptr()] = self
    init = optim._Table.__init__

    def call(name, *args):
        t = tables.get(args[1]) if name in ("bts_adamw_multi_step", "bts_adamw_multi_moments") else None
        launches.append((name, None, None) if t is None else (name, t.records.numpy().copy().view(optim._RECORD), t.chunks.numpy().copy()))
        return 16384 if name == "bts_adamw_multi_workspace_bytes" else 0
    for name, value in (("call", call), ("require_gpu", lambda t: None), ("current_device", lambda: None), ("raw_stream", lambda: 0)):
        monkeypatch.setattr(optim, name, value)
    monkeypatch.setattr(optim._Table, "__init__", table)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: 0)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, s: None)
    monkeypatch.setattr(torch, "empty", lambda *a, pin_memory=False, **kw: empty(*a, **kw))
    return launches


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_sees_a_parameter_that_shrinks_in_place(stubbed_adamw, bits):
    """p.data = p.data[:k] keeps the address and, for a vector, the stride: a launch with the old length would read behind the new gradient."""
    from bts_amd.optim import FusedAdamW
    p, q = torch.nn.Parameter(torch.zeros(9000)), torch.nn.Parameter(torch.zeros(50))
    opt = FusedAdamW([p, q], state_bits=bits)
    p.grad, q.grad = torch.zeros(9000), torch.zeros(50)
    opt.step()
    assert stubbed_adamw[-1][1]["n"].tolist() == [9000, 50]
    p.grad = torch.zeros(9000)                                  # a gradient elsewhere: the same table, its address in it
    opt.step()
    assert stubbed_adamw[-1][1]["g"].tolist() == [p.grad.data_ptr(), q.grad.data_ptr()]
    opt.moments()
    n = len(stubbed_adamw)
    p.data = p.data[:5000]
    for grad in (torch.zeros(5000), None):                      # a new gradient; none set anew: the old one, of 9000 elements
        if grad is not None:
            p.grad = grad
        else:
            p.data = p.data[:4500]
        for use in (opt.step, opt.step, opt.moments):           # its state is one of 9000 elements: refused, again and again
            with pytest.raises(_lib.BtsAmdError):
                use()
    assert len(stubbed_adamw) == n
    p.data, p.grad = torch.zeros(9000), torch.zeros(9000)
    opt.step()
    assert stubbed_adamw[-1][1]["n"].tolist() == [9000, 50]
    n = len(stubbed_adamw)
    p.grad.data = torch.zeros(8000)                             # a gradient that is not the parameter's any more
    with pytest.raises(_lib.BtsAmdError):
        opt.step()
    assert len(stubbed_adamw) == n


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_memory_outlives_the_work_of_every_stream(stubbed_adamw, monkeypatch, bits):
    """Table made on one stream, used on others: everything that a launch reads and writes is recorded for the launch's stream (recording
    memory for its own stream does nothing), also after a gradient moved and the records alone were made anew."""
    from bts_amd import optim
    now, recorded = [0], set()
    monkeypatch.setattr(optim, "raw_stream", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: now[0])
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, s: recorded.add((self.untyped_storage().data_ptr(), s)))
    p, q = torch.nn.Parameter(torch.zeros(9000)), torch.nn.Parameter(torch.zeros(50))
    opt = optim.FusedAdamW([p, q], state_bits=bits, max_grad_norm=1.0)
    p.grad, q.grad = torch.zeros(9000), torch.zeros(50)

    def kept(*more):
        own = [t for st in opt.state.values() for t in st.values() if torch.is_tensor(t) and t.dim()]
        return {t.untyped_storage().data_ptr() for t in own + list(more) if t is not None}
    opt.step()
    opt.moments()
    for stream in (1, 2):
        now[0] = stream
        recorded.clear()
        p.grad = torch.zeros(9000)                              # a new copy of the records, made on this stream
        opt.step()
        mine = kept(opt._plan.chunks, opt._hyper, opt._norm, opt._scratch)
        assert mine <= {t for t, s in recorded if s == stream}
        opt.moments()
        table = opt._state_plan["table"]
        assert kept(table.chunks, table.records, table.offsets) <= {t for t, s in recorded if s == stream}
    now[0] = 1                                                  # the records of the last upload belong to stream 2
    recorded.clear()
    opt.step()
    assert (opt._plan.records.data_ptr(), 1) in recorded
    opt._hyper = None                                           # new rows, used for the first time by prepare_step on stream 3
    now[0] = 0
    opt._rows()
    now[0] = 3
    opt.prepare_step()
    assert (opt._hyper.data_ptr(), 3) in recorded


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_sees_that_a_parameter_changed_its_order_in_memory(stubbed_adamw, bits):
    """model.to(memory_format=torch.channels_last) between two steps: the codes lie in the old order."""
    from bts_amd.optim import FusedAdamW
    p = torch.nn.Parameter(torch.zeros(40, 24, 3, 3))
    opt = FusedAdamW([p], state_bits=bits)
    p.grad = torch.zeros_like(p)
    opt.step()
    opt.moments()
    p.data = p.data.contiguous(memory_format=torch.channels_last)
    p.grad = torch.zeros_like(p)
    n = len(stubbed_adamw)
    with pytest.raises(_lib.BtsAmdError, match="load_state_dict"):
        opt.step()
    assert len(stubbed_adamw) == n
    assert all(t.shape == p.shape and t.is_contiguous() for t in opt.moments()[0])       # the values where they belong
    p.data = torch.zeros(40, 24, 3, 3)
    p.grad = torch.zeros_like(p)
    opt.step()
    assert stubbed_adamw[-1][0] == "bts_adamw_multi_step"


def test_adamw_captured_steps_keep_the_memory_of_parameters_and_gradients(stubbed_adamw, monkeypatch):
    """A graph goes on writing the addresses that it was captured with, also after p.data was given other memory."""
    from bts_amd.optim import FusedAdamW
    p = torch.nn.Parameter(torch.zeros(5000))
    opt = FusedAdamW([p], state_bits=8)
    p.grad = torch.zeros(5000)
    opt.step()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    opt.step(prepared=True)
    rec = stubbed_adamw[-1][1]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    p.data, p.grad.data = torch.zeros(5000), torch.zeros(5000)
    p.grad = None

    def tensors(x):
        return [x] if torch.is_tensor(x) else [t for y in x for t in tensors(y)] if isinstance(x, (list, tuple)) else []
    kept = {t.data_ptr() for t in tensors(opt._kept)}
    assert {int(rec["p"][0]), int(rec["g"][0]), int(rec["m"][0]), int(rec["v"][0])} <= kept


@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode_derivatives_are_refused(stubbed_norm, needs_grad):
    import torch.autograd.forward_ad as forward_ad
    x, w, b = torch.randn(3, 8), torch.ones(8), torch.zeros(8)
    w.requires_grad_(needs_grad)
    with forward_ad.dual_level():
        assert layer_norm(x, w, b).shape == x.shape                       # no tangent anywhere: nothing is lost
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for i in range(3):
                    args = [x, w.detach(), b]
                    args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                    with pytest.raises(NotImplementedError):
                        layer_norm(*args)
    n = len(stubbed_norm)
    assert layer_norm(x, w.detach(), b).shape == x.shape and len(stubbed_norm) == n + 1


@pytest.mark.parametrize("needs_grad", [False, True])
def test_tracing_is_refused(stubbed_norm, needs_grad):
    with pytest.raises(_lib.BtsAmdError, match="traced"):
        torch.jit.trace(LayerNorm(8).requires_grad_(needs_grad), torch.randn(3, 8), check_trace=False)
    assert not stubbed_norm and LayerNorm(8)(torch.randn(3, 8)).shape == (3, 8)


@pytest.mark.parametrize("kw", [dict(state_bits=8), dict(state_bits=32), dict()])
def test_adamw_a_refused_checkpoint_changes_nothing(stubbed_adamw, kw):
    import copy
    from bts_amd.optim import FusedAdamW
    p, q = torch.nn.Parameter(torch.zeros(5000)), torch.nn.Parameter(torch.zeros(50))
    opt = FusedAdamW([{"params": [p, q], "lr": 0.5}], **kw)
    if kw:
        p.grad, q.grad = torch.zeros(5000), torch.zeros(50)
        opt.step()
        good = opt.state_dict()
    else:                                                       # (its step has no form without a GPU)
        good = {"state": {i: {"step": torch.tensor(1.0), "exp_avg": torch.zeros(n), "exp_avg_sq": torch.zeros(n)} for i, n in ((0, 5000), (1, 50))},
                "param_groups": opt.state_dict()["param_groups"]}
        opt.load_state_dict(good)
    had = {id(t): {k: v for k, v in st.items()} for t, st in opt.state.items()}
    hyper = opt._hyper
    bads = [lambda sd: sd["state"][1].update(step=torch.tensor(7.0))]
    bads += [lambda sd: sd["state"][1].update(exp_avg=torch.zeros(3)), lambda sd: sd["state"][0].pop("exp_avg_sq")]
    bads += [lambda sd: sd["state"][1].pop("step")] if kw else []
    for bad in bads:
        sd = copy.deepcopy(good)
        sd["param_groups"][0]["lr"] = 0.25
        bad(sd)
        with pytest.raises(_lib.BtsAmdError):
            opt.load_state_dict(sd)
        assert opt.param_groups[0]["lr"] == 0.5 and opt._hyper is hyper
        assert {id(t): set(st) for t, st in opt.state.items()} == {t: set(st) for t, st in had.items()}
        assert all(st[k] is had[id(t)][k] for t, st in opt.state.items() for k in st if k != "step")
    with pytest.raises(ValueError):                             # torch's own refusal
        opt.load_state_dict({"state": {}, "param_groups": []})
    if kw:
        opt.step()
        assert stubbed_adamw[-1][0] == "bts_adamw_multi_step"


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_sees_that_states_were_reset(stubbed_adamw, bits):
    from collections import defaultdict
    from bts_amd.optim import FusedAdamW
    ps = [torch.nn.Parameter(torch.zeros(n)) for n in (5000, 50, 6000)]
    opt = FusedAdamW(ps, state_bits=bits)
    for p in ps:
        p.grad = torch.zeros_like(p)

    def step():
        opt.step()
        rec = stubbed_adamw[-1][1]
        opt.moments()
        seen = stubbed_adamw[-1][1]
        own = [opt.state[p]["exp_avg_codes" if "exp_avg_codes" in opt.state[p] else "exp_avg"].data_ptr() for p in ps]
        assert rec["m"].tolist() == seen["m"].tolist() == own and set(opt.state_dict()["state"]) == {0, 1, 2}
        return [opt.state[p] for p in ps]
    first = step()
    assert all(a is b for a, b in zip(first, step()))
    opt.state = defaultdict(dict)
    second = step()
    assert not any(a is b for a, b in zip(first, second))
    opt.state[ps[1]] = {}
    third = step()
    assert [a is b for a, b in zip(second, third)] == [True, False, True]
    opt.state.pop(ps[2])
    fourth = step()
    opt.state[ps[0]].clear()
    step()
    opt.state.clear()
    assert not any(a is b for a, b in zip(fourth, step()))
    opt.state.clear()
    assert all((t == 0).all() for mv in opt.moments() for t in mv) and not opt.state_dict()["state"]
    ps[0].data = ps[0].data[:10]                                # a parameter without a state
    assert [m.numel() for m, _ in opt.moments()] == [10, 50, 6000] and opt.moments(flat=True)[0].numel() == 6060


def test_parameters_of_another_shape_are_refused_before_the_launch(monkeypatch):
    """[1, C] has C elements, but its gradient would come back as [C]."""
    monkeypatch.setattr(_lib, "require_gpu", lambda t: None)
    monkeypatch.setattr(ops, "current_device", lambda: -1)
    monkeypatch.setattr(ops, "raw_stream", lambda: 0)
    launches = []
    monkeypatch.setattr(ops, "call", lambda *a: launches.append(a[0]))
    x = torch.randn(3, 8)
    for shape in ((1, 8), (8, 1), (2, 4), (7,), ()):
        for args in ((torch.ones(shape), torch.zeros(8)), (torch.ones(8), torch.zeros(shape)), (torch.ones(shape).requires_grad_(True), None)):
            with pytest.raises(_lib.BtsAmdError, match="vector"):
                layer_norm(x, *args)
    assert not launches
    layer_norm(x, torch.ones(8), torch.zeros(8))
    LayerNorm((2, 4))(x.view(3, 2, 4))
    assert launches == ["bts_layernorm_fwd"] * 2


def test_adamw_steps_without_gradients_are_not_forgotten(stubbed_adamw, monkeypatch):
    import contextlib
    import copy
    from bts_amd import optim
    p = torch.nn.Parameter(torch.zeros(50))
    opt = optim.FusedAdamW([p], state_bits=8)
    opt.step()                                                  # no gradient: no state, but the count goes on
    opt.step()
    assert opt.device_steps() == [2.0] and copy.deepcopy(opt).device_steps() == [2.0]
    opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3))]})
    opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3))]})
    assert opt.device_steps() == [2.0, 0.0, 0.0]
    opt.step()
    assert opt.device_steps() == [3.0, 1.0, 1.0] and copy.deepcopy(opt).device_steps() == [3.0, 1.0, 1.0]
    sd = opt.state_dict()
    sd["state"] = {0: {"step": torch.tensor(8.0), "exp_avg": torch.zeros(50), "exp_avg_sq": torch.zeros(50)}}
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    opt.load_state_dict(sd)                                     # what a checkpoint says counts
    assert opt.device_steps() == [8.0, 0.0, 0.0]


def test_adamw_bytes_that_the_profiler_is_told(stubbed_adamw, monkeypatch):
    from bts_amd import optim
    notes = {}
    monkeypatch.setattr(optim.profiler, "ACTIVE", object())
    monkeypatch.setattr(optim.profiler, "note", lambda name, kind, work, *a: notes.update({name: work}))
    for kw, step, moments in ((dict(state_bits=8), 5000 * 16 + 50 * 28 + 6000 * 10, 11000 * 10 + 50 * 16), (dict(state_bits=32), 5050 * 28 + 6000 * 22, 11050 * 16),
                              (dict(state_bits=8, max_grad_norm=1.0), 5000 * 20 + 50 * 32 + 6000 * 12, 11000 * 10 + 50 * 16)):
        ps = [torch.nn.Parameter(torch.zeros(n, dtype=t)) for n, t in ((5000, torch.float32), (50, torch.float32), (6000, torch.bfloat16), (7000, torch.float32))]
        for p in ps[:3]:                                        # the last one has no gradient, no state and no part
            p.grad = torch.zeros_like(p)
        opt = optim.FusedAdamW(ps, **kw)
        opt.step()
        opt.moments()
        assert notes == {"adamw_multi_step": step, "adamw_moments": moments}


def test_adamw_captured_work_keeps_the_device_rows(stubbed_adamw, monkeypatch):
    """A captured step without gradients, or a captured prepare_step, writes the rows, too: add_param_group makes them anew."""
    from bts_amd.optim import FusedAdamW
    for use in (lambda o: o.step(prepared=True), lambda o: o.prepare_step()):
        opt = FusedAdamW([torch.nn.Parameter(torch.zeros(50))], max_grad_norm=1.0)
        opt.step()
        with monkeypatch.context() as m:
            m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
            use(opt)
        rows, norm = opt._hyper.data_ptr(), opt._norm.data_ptr()
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3))]})
        kept = {t.data_ptr() for k in opt._kept for t in k if torch.is_tensor(t)}
        assert {rows, norm} <= kept


def test_the_gpu_tests_reach_every_kernel():
    """Forward and backward are compared with the definition for every variant (lanes, vectors a lane, odd widths), and with a block that
    walks several rows for every variant of odd widths that has more than one vector a row."""
    from tests.test_gpu_6_layer_norm import MORE, SHAPES

    def variant(vec, c):                                        # the launcher's rule
        nv = -(-c // vec)
        most = 1 if nv <= 64 else (16 if c <= 1024 or c > 8192 else 8) // vec
        lanes = 1
        while lanes * most < nv:
            lanes *= 2
        if nv > 64:
            lanes = 64 if c <= 1024 else -(-nv // 64) * 64 if vec == 8 and nv <= 384 else max(lanes, 256)
        return lanes, -(-nv // lanes), c % vec != 0
    for dtype, vec in ((torch.float32, 4), (torch.bfloat16, 8)):
        cases = SHAPES + [(m, c) for t, m, c in MORE if t == dtype]
        every = {variant(vec, c) for c in range(1, ops.LN_MAX_C + 1)}
        assert every == {variant(vec, c) for _, c in cases}
        walked = {}
        for m, c in cases:
            lanes, _, odd = variant(vec, c)
            rows = 256 * (1024 // lanes if lanes > 64 else 4 * (256 // lanes))         # of a whole grid of the backward pass with sums
            if odd and lanes >= 64 and m > rows:
                walked[variant(vec, c)[:2]] = m
        missing = {v[:2] for v in every if v[2] and v[0] >= 64} - set(walked)
        assert not missing, (dtype, missing)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_a_reset_state_takes_the_parameters_new_shape(stubbed_adamw, bits):
    from bts_amd.optim import FusedAdamW
    p, q = torch.nn.Parameter(torch.zeros(9000)), torch.nn.Parameter(torch.zeros(50))
    opt = FusedAdamW([p, q], state_bits=bits)
    p.grad, q.grad = torch.zeros(9000), torch.zeros(50)
    opt.step()
    opt.moments()
    p.data, p.grad = p.data[:5000], None
    p.grad = torch.zeros(5000)
    with pytest.raises(_lib.BtsAmdError):
        opt.step()
    opt.state[p] = {}
    opt.step()
    assert stubbed_adamw[-1][1]["n"].tolist() == [5000, 50] and [m.numel() for m, _ in opt.moments()] == [5000, 50]
    assert opt.moments(flat=True)[0].numel() == 5050 and stubbed_adamw[-1][1]["n"].tolist() == [5000, 50]


def test_adamw_sees_a_parameter_transposed_in_place(stubbed_adamw):
    """p.data = p.data.t() keeps address and size; a contiguous gradient of the new shape lies in another order."""
    from bts_amd.optim import FusedAdamW
    p = torch.nn.Parameter(torch.zeros(60, 80))
    opt = FusedAdamW([p], state_bits=8, min_8bit_size=1)
    p.grad = torch.zeros(60, 80)
    opt.step()
    p.data, p.grad = p.data.t(), None
    n = len(stubbed_adamw)
    for grad in (torch.zeros(80, 60), torch.zeros(60, 80).t()):
        p.grad = grad
        with pytest.raises(_lib.BtsAmdError):
            opt.step()
    assert len(stubbed_adamw) == n


def test_backward_refuses_what_comes_back_on_another_device(stubbed_norm, monkeypatch):
    """(Stand-ins for a GPU: the gradient claims device 0, and so does what the forward pass saved.)"""
    moved, keep = set(), []
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: -1 if t.data_ptr() in moved else 0)
    monkeypatch.setattr(ops, "current_device", lambda: 0)

    def refuse(t):
        raise _lib.BtsAmdError("not on a GPU")
    monkeypatch.setattr(_lib, "require_gpu", refuse)

    def move(t):
        keep.append(t.clone())
        moved.add(keep[-1].data_ptr())
        return keep[-1]
    for only in ((8, 16), (16,)):
        x, w = torch.randn(8, 16, requires_grad=True), torch.ones(16, requires_grad=True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: move(t) if t.shape == only else t):
            y = layer_norm(x, w)
        n = len(stubbed_norm)
        with pytest.raises(_lib.BtsAmdError):
            y.sum().backward()
        assert len(stubbed_norm) == n


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_refuses_states_on_another_device(stubbed_adamw, bits):
    """An optimizer whose state tensors were moved off the device: a new table must not take their addresses."""
    from bts_amd.optim import FusedAdamW
    for k in (("exp_avg_codes", "exp_avg_scales", "exp_avg_sq_codes", "exp_avg_sq_scales") if bits == 8 else ("exp_avg", "exp_avg_sq")):
        p = torch.nn.Parameter(torch.zeros(9000))
        opt = FusedAdamW([p], state_bits=bits)
        p.grad = torch.zeros(9000)
        opt.step()
        opt.state[p] = {**opt.state[p], k: opt.state[p][k].to("meta")}
        n = len(stubbed_adamw)
        for use in (opt.step, opt.moments):
            with pytest.raises(_lib.BtsAmdError):
                use()
        assert len(stubbed_adamw) == n
