"""Fused multi-tensor AdamW on the HIP kernels `bts_adamw_advance` + `bts_adamw_step`.

Semantics and state layout of ``torch.optim.AdamW`` (bts_main.py:371-373): per-parameter state
``{'step', 'exp_avg', 'exp_avg_sq'}``, index-keyed ``state_dict()``, so optimizer checkpoints written by
the reference's AdamW load here and vice versa (bts_main.py:383-387, 498-503).  One kernel launch per
parameter group replaces the per-tensor update chain.

The step count lives on the DEVICE, one 8-float row per parameter group
(``{lr, bias_c1, bias_c2, step, beta1, beta2, -, -}``): ``bts_adamw_advance`` increments it and refreshes the bias
corrections in front of the update kernels, so a captured hipGraph advances the optimizer on every replay with no
host involvement.  The host only rewrites ``lr`` (the per-step poly schedule, bts_main.py:456-458: ``prepare_step``)
and reads ``step`` back when a checkpoint is written (``state_dict``); ``load_state_dict`` restores the counter
from the checkpoint's per-parameter ``step``, so resumed training continues with the right bias corrections.

Restriction (documented, checked): the step count is ONE value per parameter group, where ``torch.optim.AdamW`` keeps one per
parameter.  The two coincide whenever every parameter of a group receives a gradient on every step -- the case of
bts_main.py, where frozen parameters are filtered out before the groups are built.  ``load_state_dict`` refuses a checkpoint
whose per-parameter steps differ inside a group instead of silently rewriting them, and ``step(closure)`` is not supported.

Gradients must keep their storage between steps (call ``zero_grad(set_to_none=False)``, the default here):
the device pointer tables are rebuilt only when a pointer changes.

Options beyond that, all on `bts_adamw_multi_step` (csrc/adamw.hip; one update launch for ALL groups):

* ``state_bits=32``: f32 moments as without it, every constant formed in 64 bits.  (`bts_adamw_step`, which f32 parameters take when no option
  is given, forms 1 - beta2 in f32: its exp_avg_sq is 4.7e-5 of itself larger for beta2 = 0.999, and bias_c2 with it, so the updates agree.)
* ``state_bits=8``: the moments of parameters with at least ``min_8bit_size`` elements are held as 8-bit codes, 256 elements (in the
  parameter's memory order) to a power of two: 2 bytes of state per element instead of 8, read and written once per step.  Codes and
  scales are ``state[p]['exp_avg_codes' / 'exp_avg_scales' / 'exp_avg_sq_codes' / 'exp_avg_sq_scales']``; ``moments()`` gives the values that
  they stand for.  Shorter parameters keep 32 bits.  ``state_dict()`` is torch.optim.AdamW's with the f32 values, and loading such a
  state -- from here, or from the reference's optimizer -- forms the codes again: values that came from codes give the same values.
* ``max_grad_norm``: the gradients of all groups are scaled by min(1, max_grad_norm / (norm + 1e-6)) inside the step, where norm is their
  common 2-norm (torch.nn.utils.clip_grad_norm_'s rule; the gradients themselves stay as they are).  No host synchronisation:
  ``grad_norm`` is a device tensor that every step rewrites.  ``float('inf')`` only measures: gradients that are not finite stay
  their own elements' matter, where a finite bound makes every parameter NaN for a norm that is (clip_grad_norm_'s rule).
* bf16 parameters (with bf16 gradients; states stay f32 or 8-bit, the update is formed in f32 and rounded once).

There, the tensors of a state are replaced through ``load_state_dict`` only (a state may be reset: ``opt.state = defaultdict(dict)``,
``opt.state[p] = {}``), and the learning rate is a launch argument: a captured step takes ``prepared=True`` and ``prepare_step()`` outside the
graph, as above.  A captured step works on the parameters' memory, gradients, states and step counts that it was captured with, and the
optimizer keeps them: capture again after ``load_state_dict`` or ``add_param_group``.
"""
import ctypes as C
import itertools
import math
from operator import attrgetter, is_, itemgetter

import numpy as np
import torch

from . import profiler
from ._lib import BtsAmdError, call, current_device, raw_stream, require_gpu, stream_ptr

_ROW = 8        # floats per group row (include/bts_amd.h: bts_adamw_advance)
_WIDE_ROW = 16  # doubles per group row of bts_adamw_multi_step (BTS_ADAMW_ROW)
_CHUNK, _BLOCK, _MAX_GROUPS = 4096, 256, 64
_BF16, _8BIT = 1, 2
_RECORD = np.dtype([("p", "u8"), ("g", "u8"), ("m", "u8"), ("v", "u8"), ("m_scale", "u8"), ("v_scale", "u8"), ("n", "i8"), ("group", "i4"), ("flags", "i4")])
_RUN_FIRST = "run one step with the same parameters and gradients (zero_grad(set_to_none=False) keeps them)"
_CODES = ("exp_avg_codes", "exp_avg_scales", "exp_avg_sq_codes", "exp_avg_sq_scales")
_ptr, _stride, _numel, _grad, _dtype = torch.Tensor.data_ptr, torch.Tensor.stride, torch.Tensor.numel, attrgetter("grad"), attrgetter("dtype")
_contiguous, _params = torch.Tensor.is_contiguous, itemgetter("params")


def _dense(t):
    """Every element of t's storage span belongs to t once (any order of dimensions)."""
    if t.is_contiguous():
        return True
    expect = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if st != expect:
            return False
        expect *= n
    return True


def _room(t):
    """Bytes of t's storage from t's first element on."""
    return t.untyped_storage().nbytes() - t.storage_offset() * t.element_size()


def _same_strides(a, b, shape):
    return a == b or all(x == y for x, y, n in zip(a, b, shape) if n != 1)           # (a size-1 dimension's stride is free)


def _same_layout(t, p):
    return _same_strides(t.stride(), p.stride(), p.shape)


def _layout(t):
    return t.size(), t.stride()


def _layout_of(st, p):
    """Shape and order in memory that p's state `st` was made for."""
    return _layout(p) if not st else st["layout"] if "layout" in st else _layout(st["exp_avg"])


def _like(flat, off, layout):
    """The elements of `flat` from `off` on, with the shape and order in memory of _layout(p)."""
    return torch.as_strided(flat, *layout, flat.storage_offset() + off)


class _Table:
    """Device tables of one list of tensors: records and chunks of bts_adamw_multi_*, and what they were made from."""

    def __init__(self, records, sizes, device):
        counts = np.array([-(-n // _CHUNK) for n in sizes], dtype=np.int64)
        self.n_chunks = int(counts.sum())
        chunks = np.empty((self.n_chunks, 2), dtype=np.int32)
        chunks[:, 0] = np.repeat(np.arange(len(sizes), dtype=np.int32), counts)
        chunks[:, 1] = np.arange(self.n_chunks) - np.repeat(np.cumsum(counts) - counts, counts)
        self.host = records
        self.holds = self.offsets = None        # what must live as long as the addresses; begin of each tensor in flat moments
        self.states = self.shaped = None        # _states_now() when it was made; the parameters that have an order in memory
        self.chunks = torch.from_numpy(chunks).to(device)
        self.records = torch.from_numpy(records.view(np.uint8)).to(device)
        self.records_on, self.used_on = raw_stream(), set()

    def upload(self, device):
        """A new device copy of the records, without waiting for it: launches in flight may still read the old one."""
        pinned = torch.empty(self.host.nbytes, dtype=torch.uint8, pin_memory=True)
        pinned.numpy()[:] = self.host.view(np.uint8)
        self.records = pinned.to(device, non_blocking=True)
        self.records_on = raw_stream()

    def use(self, stream, states_on):
        """Called before a launch on `stream`, the current one: memory that the allocator gave to another one must outlive this one's work
        -- the tables, and the states that the launch writes, also where the optimizer drops them while it runs."""
        if stream not in self.used_on:
            self.used_on.add(stream)
            _record([self.chunks, self.offsets])
            if states_on != {stream}:
                _record({t.untyped_storage().data_ptr(): t for t in self.holds[1] if t.numel()}.values())
        if stream != self.records_on:
            _record([self.records])


def _record(ts):
    cur = torch.cuda.current_stream()
    for t in ts:
        if t is not None and t.numel():
            t.record_stream(cur)            # (nothing to do, and nothing done, for memory of the current stream)


class FusedAdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=None, max_grad_norm=None, min_8bit_size=4096):
        if state_bits not in (8, 32, None):
            raise BtsAmdError("FusedAdamW: state_bits must be 8, 32 or None, got %r" % (state_bits,))
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise BtsAmdError("FusedAdamW: max_grad_norm must be positive (or None), got %r" % (max_grad_norm,))
        if int(min_8bit_size) != min_8bit_size or min_8bit_size < 1:
            raise BtsAmdError("FusedAdamW: min_8bit_size must be a positive whole number, got %r" % (min_8bit_size,))
        self._options = (state_bits or 32, int(min_8bit_size), None if max_grad_norm is None else float(max_grad_norm))
        self._multi = state_bits is not None or max_grad_norm is not None
        self._forget()
        self._states_on = set()
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        super().__init__(params, defaults)

    # the options are the constructor's: the layout of states and device rows goes by them
    state_bits = property(lambda self: self._options[0])
    min_8bit_size = property(lambda self: self._options[1])
    max_grad_norm = property(lambda self: self._options[2])

    def _forget(self):
        self._tables = {}
        self._hyper = None          # [n_groups, 8] f32 on the device (bts_adamw_step), or [n_groups + 1, 16] f64 (bts_adamw_multi_step)
        self._seen = self._plan = self._state_plan = None
        self._steps = None          # step counts of the groups while there are no device rows, where the states do not say them
        self._kept = []             # what captured graphs refer to
        self._scratch = self._norm = None
        self._used_on = set()       # streams that _hyper, _scratch and _norm are recorded for
        self._states_on = {None}    # streams that the states were allocated on; None: who knows

    def __getstate__(self):         # copies and pickles: states with their step counts, nothing that holds addresses
        self._refresh_steps()
        return {**super().__getstate__(), "_options": self._options, "_multi": self._multi, "_steps": self.device_steps()}

    def __setstate__(self, state):  # (load_state_dict calls it too, with the loaded states and groups)
        super().__setstate__(state)
        if "_options" in state:
            self._forget()
            self._steps = state.get("_steps")

    def add_param_group(self, param_group):
        old = getattr(self, "_hyper", None)
        if old is not None:         # the device rows have one row per group: keep their step counts, make them anew
            self._refresh_steps()
            self._steps = self.device_steps()
            self._hyper = None
        super().add_param_group(param_group)
        self._seen = None
        if not self._multi and any(p.dtype != torch.float32 for p in self.param_groups[-1]["params"]):
            self._multi, self._tables, self._states_on = True, {}, {None}

    # ---- device-resident schedule / step counter ------------------------------------------------
    def _device(self):
        for g in self.param_groups:
            for p in g["params"]:
                return p.device
        raise BtsAmdError("FusedAdamW has no parameters")

    def _elsewhere(self):
        """The parameters' device if it is not the current one (launches and streams go by the current device)."""
        for g in self.param_groups:
            for p in g["params"]:
                require_gpu(p)
                return None if p.device.index == current_device() else p.device
        raise BtsAmdError("FusedAdamW has no parameters")

    def _group_step_from_state(self, g):
        """Step count recorded in the per-parameter state of group g (0 if the group has no state yet)."""
        seen = set()
        for p in g["params"]:
            st = self.state.get(p)
            if st and "step" in st:
                seen.add(float(st["step"]))
        return self._one_step(seen)

    @staticmethod
    def _one_step(seen):
        if len(seen) > 1:
            raise BtsAmdError("FusedAdamW keeps one step count per parameter group; this state has steps %s inside one group "
                              "(load it with torch.optim.AdamW, or regroup the parameters)" % sorted(seen))
        return seen.pop() if seen else 0.0

    def _group_steps(self):
        """Step counts without device rows: carried over from earlier ones (a group that took steps without gradients has no state to say
        it), else what the states say."""
        known = self._steps or []
        return [known[gi] if gi < len(known) else self._group_step_from_state(g) for gi, g in enumerate(self.param_groups)]

    def _rows(self):
        """The device rows, created on first use from the groups' hyper-parameters and recorded state."""
        if self._hyper is None:
            self._used_on = set()
            steps = self._group_steps()
            if self._multi:
                rows = np.zeros((len(self.param_groups) + 1, _WIDE_ROW))
                for r, g, t in zip(rows, self.param_groups, steps):
                    r[0], r[3], r[4:6], r[6], r[7] = float(g["lr"]), t, g["betas"], g["eps"], g["weight_decay"]
                rows[-1, 0] = math.inf if self.max_grad_norm is None else self.max_grad_norm
                self._hyper, self._steps = torch.from_numpy(rows).to(self._device()), None
                return self._hyper
            rows = []
            for g, t in zip(self.param_groups, steps):
                b1, b2 = g["betas"]
                rows.append([float(g["lr"]), 1.0, 1.0, t, float(b1), float(b2), 0.0, 0.0])
            self._hyper, self._steps = torch.tensor(rows, dtype=torch.float32).to(self._device()), None
        return self._hyper

    def _launch_on(self, table=None):
        """The current stream, for a launch that works on the rows, and on what `table` says."""
        stream = raw_stream()
        if stream not in self._used_on:
            self._used_on.add(stream)
            _record([self._hyper, self._scratch, self._norm])
        if table is not None:
            table.use(stream, self._states_on)
        if torch.cuda.is_current_stream_capturing():            # what a graph writes stays its own, whatever is made anew here
            self._kept.append((self._hyper, self._scratch, self._norm) + (() if table is None else (table.records, table.chunks, table.offsets, table.holds)))
        return stream

    def _host_hyper(self, lrs=None):
        """The groups' hyper-parameters as bts_adamw_multi_step takes them from the host."""
        vals = []
        for gi, g in enumerate(self.param_groups):
            b1, b2 = g["betas"]
            vals += [float(g["lr"] if lrs is None else lrs[gi]), float(b1), float(b2), float(g["eps"]), float(g["weight_decay"])]
        vals.append(math.inf if self.max_grad_norm is None else self.max_grad_norm)
        return (C.c_double * len(vals))(*vals)

    def prepare_step(self, lrs=None):
        """Host side of a step: write the groups' learning rates into the device rows.  Call OUTSIDE a captured
        graph (step() calls it itself unless ``prepared=True``)."""
        if self._multi and self._elsewhere() is not None:
            with torch.cuda.device(self._elsewhere()):
                return self.prepare_step(lrs)
        rows = self._rows()
        if self._multi:
            call("bts_adamw_multi_set", rows.data_ptr(), len(self.param_groups), self._host_hyper(lrs), self._launch_on())
            return
        vals = [float(g["lr"] if lrs is None else lrs[gi]) for gi, g in enumerate(self.param_groups)]
        rows[:, 0].copy_(torch.tensor(vals, dtype=torch.float32))

    def device_steps(self):
        """Per-group step counts as python floats (synchronises)."""
        if self._hyper is None:
            return self._group_steps()
        return [float(v) for v in self._hyper[:len(self.param_groups), 3].cpu()]

    def _refresh_steps(self):
        steps = self.device_steps()
        for gi, g in enumerate(self.param_groups):
            for p in g["params"]:
                st = self.state.get(p)
                if st:
                    st["step"] = torch.tensor(steps[gi], dtype=torch.float32)

    @property
    def grad_norm(self):
        """The 2-norm of all gradients of the last step (f32, on the device), None without max_grad_norm or before the first step."""
        return None if self._norm is None else self._norm[0]

    # ---- torch.optim.Optimizer surface -------------------------------------------------------------
    def zero_grad(self, set_to_none=False):
        for g in self.param_groups:
            for p in g["params"]:
                if p.grad is not None:
                    if set_to_none:
                        p.grad = None
                    else:
                        p.grad.zero_()
        if set_to_none:
            self._tables = {}

    def state_dict(self):
        """torch.optim.AdamW layout; the per-parameter ``step`` entries are refreshed from the device counter first
        (they are not touched by step(), which may be running inside a replayed graph)."""
        self._refresh_steps()
        if not (self._multi and self.state):
            return super().state_dict()
        put = self.register_state_dict_post_hook(FusedAdamW._put_moments, prepend=True)                 # before the user's hooks
        try:
            return super().state_dict()
        finally:
            put.remove()

    def _put_moments(self, sd):
        ps = [p for g in self.param_groups for p in g["params"]]
        for i, (p, (m, v)) in enumerate(zip(ps, self.moments())):
            st = self.state.get(p)
            if st:
                sd["state"][i] = {"step": st["step"], "exp_avg": m, "exp_avg_sq": v}

    def load_state_dict(self, state_dict):
        # Between the user's hooks: what their pre hooks made of the checkpoint counts, and is checked before anything changes; their post
        # hooks find the optimizer whole.
        last = []
        check = self.register_load_state_dict_pre_hook(lambda _, sd: last.append(self._check_loaded(sd)))
        rebuild = self.register_load_state_dict_post_hook(lambda _: self._loaded(last[-1]), prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            check.remove()
            rebuild.remove()

    def _loaded(self, state_dict):
        # the moment buffers were replaced and the step count comes from the checkpoint: drop every cached pointer
        # table and rebuild the device rows (step, betas, lr) from what was just loaded
        self._tables = {}
        self._hyper = self._seen = self._plan = self._state_plan = self._steps = None
        if self._multi:
            self._load_moments(state_dict)
        else:
            for p, st in self.state.items():        # the kernel walks parameter and moments with one index: same order in memory
                for k in ("exp_avg", "exp_avg_sq"):
                    if k in st and st[k].stride() != p.stride():
                        st[k] = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(st[k])
        self._rows()

    def _check_loaded(self, state_dict):
        """Refuses a checkpoint that does not fit while this optimizer is still whole."""
        saved = state_dict["param_groups"]
        if [len(g["params"]) for g in saved] != [len(g["params"]) for g in self.param_groups]:
            return state_dict                       # (refused by what comes next)
        todo = []
        for g, sg in zip(self.param_groups, saved):
            there = [(i, p, state_dict["state"][i]) for i, p in zip(sg["params"], g["params"]) if state_dict["state"].get(i)]
            self._one_step({float(st["step"]) for _, _, st in there if "step" in st})
            todo += there
        for i, p, st in todo:
            if self._multi and "step" not in st or any(k not in st or tuple(st[k].shape) != tuple(p.shape) for k in ("exp_avg", "exp_avg_sq")):
                raise BtsAmdError("FusedAdamW.load_state_dict: parameter %r needs step, and exp_avg and exp_avg_sq of shape %s" % (i, tuple(p.shape)))
        if self._multi and todo:
            self._check_parameters([p for _, p, _ in todo])
        return state_dict

    # ---- 8-bit / multi-tensor form -------------------------------------------------------------------
    def _load_moments(self, state_dict):
        ps = [p for g in self.param_groups for p in g["params"]]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        self.state.clear()
        self._states_on = set()
        todo = [(p, state_dict["state"][i]) for i, p in zip(ids, ps) if state_dict["state"].get(i)]
        if not todo:
            return
        with torch.cuda.device(self._device()):
            self._new_state([p for p, _ in todo])
            for p, st in todo:
                self.state[p]["step"] = torch.as_tensor(st["step"], dtype=torch.float32).reshape(()).cpu().clone()
            plan = self._state_table()
            table = plan["table"]
            m = torch.empty(plan["total"], dtype=torch.float32, device=self._device())
            v = torch.empty_like(m)
            torch._foreach_copy_([_like(t, plan["at"][id(p)], _layout(p)) for t in (m, v) for p, _ in todo], [st[k] for k in ("exp_avg", "exp_avg_sq") for _, st in todo])
            if table.n_chunks:
                call("bts_adamw_multi_moments", table.records.data_ptr(), table.chunks.data_ptr(), table.n_chunks, table.offsets.data_ptr(),
                     m.data_ptr(), v.data_ptr(), 1, raw_stream())

    def _check_parameters(self, ps):
        dev = ps[0].device
        require_gpu(ps[0])
        if len({id(p) for p in ps}) != len(ps):
            raise BtsAmdError("FusedAdamW: a parameter appears twice")
        if len(self.param_groups) > _MAX_GROUPS:
            raise BtsAmdError("FusedAdamW: at most %d parameter groups" % _MAX_GROUPS)
        spans = []
        for p in ps:
            if p.device != dev or p.dtype not in (torch.float32, torch.bfloat16) or p.layout != torch.strided or not _dense(p):
                raise BtsAmdError("FusedAdamW needs dense f32 or bf16 parameters on one device, got %s %s %s with strides %s" % (
                    tuple(p.shape), p.dtype, p.device, p.stride() if p.layout == torch.strided else p.layout))
            if p.numel():
                spans.append((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()))
        spans.sort()
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise BtsAmdError("FusedAdamW: two parameters overlap in memory")

    def _is_8bit(self, p):
        return self.state_bits == 8 and p.numel() >= self.min_8bit_size

    def _new_state(self, ps):
        """Zero states for parameters that have none: one allocation for all codes, one for all scales, one for all f32 moments."""
        eight, wide = [p for p in ps if self._is_8bit(p)], [p for p in ps if not self._is_8bit(p)]
        dev = self._device()
        self._states_on.add(raw_stream())
        blocks = [-(-p.numel() // _BLOCK) for p in eight]
        codes = torch.zeros((2, sum(blocks) * _BLOCK), dtype=torch.uint8, device=dev)
        scales = torch.full((2, sum(blocks)), 2.0 ** -126, dtype=torch.float32, device=dev)
        moments = torch.zeros((2, sum(p.numel() for p in wide)), dtype=torch.float32, device=dev)
        at = 0
        for p, nb in zip(eight, blocks):
            n = p.numel()
            self.state[p] = {"step": torch.zeros((), dtype=torch.float32), "exp_avg_codes": codes[0, at * _BLOCK:at * _BLOCK + n],
                             "exp_avg_scales": scales[0, at:at + nb], "exp_avg_sq_codes": codes[1, at * _BLOCK:at * _BLOCK + n],
                             "exp_avg_sq_scales": scales[1, at:at + nb], "layout": _layout(p)}
            at += nb
        at = 0
        for p in wide:
            self.state[p] = {"step": torch.zeros((), dtype=torch.float32), "exp_avg": _like(moments[0], at, _layout(p)), "exp_avg_sq": _like(moments[1], at, _layout(p))}
            at += p.numel()

    def _state_tensors(self, ps):
        return [t for p in ps for k, t in self.state[p].items() if k not in ("step", "layout")]

    def _parameters(self):
        return list(itertools.chain.from_iterable(map(_params, self.param_groups)))

    def _same_order(self, gs):
        """Parameters and gradients lie in memory as they did when the step's table was made (strides: only where some are not contiguous)."""
        if self._order is not None:
            return list(map(_stride, gs)) == self._order
        return all(map(_contiguous, gs)) and all(map(_contiguous, self._plan.shaped))

    def _states_now(self):
        return self.state, list(self.state.values()), [st for st in self.state.values() if st]

    def _same_states(self, then):
        """The states are the dicts that they were, and none was emptied."""
        state, dicts, filled = then
        return self.state is state and len(state) == len(dicts) and all(map(is_, state.values(), dicts)) and all(filled)

    def _records(self, ps, groups, as_now):
        """Rows of a device table, without the gradients' addresses: what the kernels go by is checked here.  as_now: the states must have
        been made for the shape and the order in memory that the parameters have now."""
        rows = []
        for p, gi in zip(ps, groups):
            st, n = self.state[p], p.numel()
            made, now = _layout_of(st, p), _layout(p)
            if as_now and made != now and (made[0] != now[0] or not _same_strides(made[1], now[1], now[0])):
                raise BtsAmdError("FusedAdamW: a parameter is %s with strides %s now, its state was made for %s with strides %s -- "
                                  "load_state_dict(state_dict()) makes it anew" % (tuple(now[0]), now[1], tuple(made[0]), made[1]))
            flags = _BF16 if p.dtype == torch.bfloat16 else 0
            if "exp_avg_codes" in st:
                a, sa, b, sb = (st[k] for k in _CODES)
                if not (a.dtype == b.dtype == torch.uint8 and sa.dtype == sb.dtype == torch.float32 and a.is_contiguous() and b.is_contiguous()
                        and sa.is_contiguous() and sb.is_contiguous() and a.device == b.device == sa.device == sb.device == p.device
                        and a.data_ptr() % 4 == 0 and b.data_ptr() % 4 == 0 and a.numel() == b.numel() == n
                        and sa.numel() == sb.numel() == -(-n // _BLOCK) and _room(a) >= sa.numel() * _BLOCK and _room(b) >= sa.numel() * _BLOCK):
                    raise BtsAmdError("FusedAdamW: the 8-bit state of a parameter of %d elements was replaced by something else, or is one of %d elements" % (n, a.numel()))
                rows.append((p.data_ptr(), 0, a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), n, gi, flags | _8BIT))
            else:
                a, b = st["exp_avg"], st["exp_avg_sq"]
                for t in (a, b):
                    if t.dtype != torch.float32 or t.device != p.device or t.numel() != n or not _dense(t) or t.shape != a.shape or not _same_layout(t, a):
                        raise BtsAmdError("FusedAdamW: the state of a parameter of %d elements was replaced by something else, or is one of %d elements" % (n, t.numel()))
                rows.append((p.data_ptr(), 0, a.data_ptr(), b.data_ptr(), 0, 0, n, gi, flags))
        return np.array(rows, dtype=_RECORD)

    def _step_table(self):
        """The table of all parameters that have a gradient now.  What it was made from is compared every step: addresses, sizes and types of
        parameters and gradients and the gradients' strides; a gradient that moved costs one small upload, anything else a new table."""
        ps, lens, keep = self._parameters(), [len(g["params"]) for g in self.param_groups], None
        gs = list(map(_grad, ps))
        try:
            gptr = list(map(_ptr, gs))
        except TypeError:                               # some have none
            keep = [i for i, g in enumerate(gs) if g is not None]
            ps, gs = [ps[i] for i in keep], [gs[i] for i in keep]
            gptr = list(map(_ptr, gs))
        if not ps:
            return None
        seen = (lens, keep, list(map(_ptr, ps)), list(map(_numel, ps)), list(map(_dtype, gs)))
        if (self._plan is not None and seen == self._seen and all(map(is_, ps, self._plan.holds[0])) and self._same_states(self._plan.states)
                and self._same_order(gs)):
            if gptr == self._gptr:
                return self._plan
            if list(map(_numel, gs)) == seen[3]:
                self._no_capture("step", _RUN_FIRST)
                self._plan.host["g"] = gptr
                self._plan.upload(self._device())
                self._gptr = gptr
                return self._plan
        groups = [gi for gi, n in enumerate(lens) for _ in range(n)]
        if keep is not None:
            groups = [groups[i] for i in keep]
        self._no_capture("step", _RUN_FIRST)
        self._check_parameters(ps)
        for p, g in zip(ps, gs):
            if g.layout != torch.strided or g.dtype != p.dtype or g.device != p.device or g.shape != p.shape or not _same_layout(g, p):
                raise BtsAmdError("FusedAdamW needs gradients of the parameter's type, shape and layout on its device: parameter %s %s %s, gradient %s %s %s" % (
                    tuple(p.shape), p.dtype, p.stride(), tuple(g.shape), g.dtype, g.stride() if g.layout == torch.strided else g.layout))
        fresh = [p for p in ps if not self.state.get(p)]
        if fresh:
            self._new_state(fresh)
            self._state_plan = None
        rec = self._records(ps, groups, True)
        rec["g"] = gptr
        self._plan = _Table(rec, [p.numel() for p in ps], self._device())
        self._plan.holds, self._plan.states = (ps, self._state_tensors(ps)), self._states_now()     # the addresses in the table stay theirs
        self._plan.shaped = [p for p in ps if p.dim() > 1]
        self._seen, self._gptr, self._order = seen, gptr, None
        if not all(map(_contiguous, itertools.chain(ps, gs))):
            self._order = list(map(_stride, gs))
        moves = 3 if self.max_grad_norm is None else 4          # parameter read and written, gradient read -- twice for its norm
        self._bytes = sum(p.numel() * (moves * p.element_size() + (4 if self._is_8bit(p) else 16)) for p in ps)
        return self._plan

    def _no_capture(self, what, how):
        if torch.cuda.is_current_stream_capturing():
            raise BtsAmdError("FusedAdamW.%s: device tables cannot be made while a graph is captured -- %s first" % (what, how))

    def _state_table(self):
        """The table of all parameters that have a state, for bts_adamw_multi_moments, and where each begins in flat moments."""
        ps, plan = self._parameters(), self._state_plan
        if (plan is None or len(ps) != len(plan["all"]) or not all(map(is_, ps, plan["all"])) or not self._same_states(plan["table"].states)
                or any(p.shape != shape for p, shape in plan["bare"])):
            self._no_capture("moments", "call moments() once")
            have = [i for i, p in enumerate(ps) if self.state.get(p)]
            hp, layouts = [ps[i] for i in have], [_layout_of(self.state.get(p), p) for p in ps]
            sizes = [math.prod(shape) for shape, _ in layouts]
            offs = [0] + list(itertools.accumulate(sizes))
            table = _Table(self._records(hp, [0] * len(hp), False), [sizes[i] for i in have], self._device())
            table.holds, table.states = (ps, self._state_tensors(hp)), self._states_now()
            table.offsets = torch.tensor([offs[i] for i in have], dtype=torch.int64).to(self._device())
            self._state_plan = {"table": table, "all": ps, "at": dict(zip(map(id, ps), offs)), "total": offs[-1], "layouts": layouts,
                                "bare": [(p, p.shape) for p in ps if not self.state.get(p)],           # without a state: zeros
                                "bytes": sum(sizes[i] * (10 if "exp_avg_codes" in self.state[ps[i]] else 16) for i in have)}
        return self._state_plan

    def moments(self, flat=False):
        """What the states stand for, in f32: a list of (exp_avg, exp_avg_sq) per parameter in the groups' order, shaped like the parameters --
        or, with flat, two vectors that hold them one after the other (each with the size and memory order that its parameter had when its state
        was made).  New memory every time; zeros where a parameter has no state yet.  To be captured into a graph it must have been called once before."""
        if self._elsewhere() is not None:
            with torch.cuda.device(self._elsewhere()):
                return self.moments(flat)
        plan = self._state_table()
        if not flat:
            for p, (shape, _) in zip(plan["all"], plan["layouts"]):
                if p.shape != shape:
                    raise BtsAmdError("FusedAdamW: a parameter is %s now, its state was made for %s" % (tuple(p.shape), tuple(shape)))
        table, total = plan["table"], plan["total"]
        new, dev = torch.zeros if plan["bare"] else torch.empty, self._device()
        m, v = new(total, dtype=torch.float32, device=dev), new(total, dtype=torch.float32, device=dev)
        if table.n_chunks:
            stream = self._launch_on(table)
            if profiler.ACTIVE is not None:
                profiler.note("adamw_moments", "hbm", float(plan["bytes"]))
            call("bts_adamw_multi_moments", table.records.data_ptr(), table.chunks.data_ptr(), table.n_chunks, table.offsets.data_ptr(),
                 m.data_ptr(), v.data_ptr(), 0, stream)
        if flat:
            return m, v
        return [(_like(m, at, how), _like(v, at, how)) for at, how in zip(plan["at"].values(), plan["layouts"])]

    def _step_multi(self, prepared):
        table = self._step_table()
        rows = self._rows()
        hyper = None if prepared else self._host_hyper()
        norm = None
        if self.max_grad_norm is not None:
            if self._norm is None:
                self._norm = torch.zeros(1, dtype=torch.float32, device=self._device())
                self._scratch = torch.empty(call("bts_adamw_multi_workspace_bytes") // 8, dtype=torch.float64, device=self._device())
                self._used_on = set()
            norm = self._norm.data_ptr()
        stream = self._launch_on(table)
        if table is None or not table.n_chunks:         # no gradient at all: the step count goes on, as bts_adamw_advance does
            if hyper is not None:
                call("bts_adamw_multi_set", rows.data_ptr(), len(self.param_groups), hyper, stream)
            rows[:len(self.param_groups), 3] += 1
            if norm is not None:
                self._norm.zero_()
            return
        if torch.cuda.is_current_stream_capturing():
            # the memory itself: a parameter or gradient that is given other memory (p.data = ...) does not take this from the graph
            self._kept.append([t.detach() for p in table.holds[0] for t in (p, p.grad)])
        if profiler.ACTIVE is not None:
            profiler.note("adamw_multi_step", "hbm", float(self._bytes))
        call("bts_adamw_multi_step", table.records.data_ptr(), table.chunks.data_ptr(), table.n_chunks, rows.data_ptr(), len(self.param_groups), hyper,
             self._scratch.data_ptr() if norm is not None else None, norm, stream)
        # parameters were updated through raw pointers: tell autograd / any version-keyed cache
        torch.autograd.graph.increment_version(table.holds[0])

    def _table(self, gi, plist):
        st = [self.state[p] for p in plist]
        key = tuple((p.data_ptr(), p.grad.data_ptr(), s["exp_avg"].data_ptr(), s["exp_avg_sq"].data_ptr())
                    for p, s in zip(plist, st))
        tb = self._tables.get(gi)
        if tb is not None and tb[0] == key:
            return tb[1]
        dev = plist[0].device

        def arr(ts):
            return torch.tensor([t.data_ptr() for t in ts], dtype=torch.int64, device=dev)
        t = dict(params=arr(plist), grads=arr([p.grad for p in plist]), m1=arr([s["exp_avg"] for s in st]),
                 m2=arr([s["exp_avg_sq"] for s in st]),
                 sizes=torch.tensor([p.numel() for p in plist], dtype=torch.int64, device=dev),
                 n=len(plist), max_size=max(p.numel() for p in plist))
        self._tables[gi] = (key, t)
        return t

    def step(self, closure=None, prepared=False):
        if closure is not None:
            raise BtsAmdError("FusedAdamW.step() does not support a closure (bts_main.py never passes one)")
        if self._multi:                 # (nothing there is an operation on a tensor that requires gradients)
            if self._elsewhere() is not None:
                with torch.cuda.device(self._elsewhere()):
                    return self._step_multi(prepared)
            return self._step_multi(prepared)
        return self._step_plain(prepared)

    @torch.no_grad()
    def _step_plain(self, prepared):
        if not prepared:
            self.prepare_step()
        rows = self._rows()
        call("bts_adamw_advance", C.c_void_p(rows.data_ptr()), len(self.param_groups), stream_ptr())
        for gi, g in enumerate(self.param_groups):
            plist = [p for p in g["params"] if p.grad is not None]
            if not plist:
                continue
            for p in plist:
                st = self.state[p]
                if not st:
                    st["step"] = torch.zeros((), dtype=torch.float32)       # refreshed by state_dict()
                    st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
                dense = p.is_contiguous() or (p.dim() == 4 and p.is_contiguous(memory_format=torch.channels_last))
                same = all(a == b for a, b, n in zip(p.grad.stride(), p.stride(), p.shape) if n != 1)     # (a size-1 dimension's stride is free)
                if not (dense and same and p.dtype == torch.float32 and p.grad.dtype == torch.float32):
                    raise RuntimeError("FusedAdamW needs dense f32 parameters with identically laid out gradients")
            t = self._table(gi, plist)
            b1, b2 = g["betas"]
            if profiler.ACTIVE is not None:      # p, g, m, v read; p, m, v written
                profiler.note("adamw_step", "hbm", 28.0 * sum(p.numel() for p in plist))
            call("bts_adamw_step", C.c_void_p(t["params"].data_ptr()), C.c_void_p(t["grads"].data_ptr()),
                 C.c_void_p(t["m1"].data_ptr()), C.c_void_p(t["m2"].data_ptr()), C.c_void_p(t["sizes"].data_ptr()),
                 t["n"], t["max_size"], 0.0, float(b1), float(b2), float(g["eps"]), float(g["weight_decay"]), 1.0, 1.0,
                 C.c_void_p(rows.data_ptr() + 4 * _ROW * gi), stream_ptr())
            # parameters were updated through raw pointers: tell autograd / any version-keyed cache
            torch.autograd.graph.increment_version(plist)
        return None
