"""Optimizers whose step is one launch of the HIP library over all parameters, with the
fp32 master -> fp16/bf16 model copy folded in.

The reference leaves the step to ``torch.optim`` (``optim.Adam`` at ``test/common.py:142,165``,
``optim.SGD`` at ``examples/tutorial.py:28``), patched by ``pyrannc/opt.py:205-312``; under amp
Apex then copies every master into its model parameter.  ``FusedAdam`` / ``FusedAdamW`` /
``FusedSGD`` keep ``torch.optim.Adam`` / ``AdamW`` / ``SGD``'s constructor arguments, parameter
groups and state layout (``step``, ``exp_avg``, ``exp_avg_sq``; ``momentum_buffer``), so state
dicts, ``patch_optimizer`` and the checkpoint slicing of ``pyrannc/opt.py:186-202`` work on
them unchanged.  There is no CPU path: parameters must live on the GPU.
"""
from __future__ import annotations

from array import array
from operator import is_
from typing import Dict, List, Optional, Tuple

import torch

from . import _lib
from .multi_tensor import _CODES, State8Plan, allocate_state8, dtype_code, stream_handle

try:        # the compiled module: lists of parameters walked in C++
    from . import _ranncgrad as _native
except ImportError:
    _native = None


_data_ptr = torch.Tensor.data_ptr
_numel = torch.Tensor.numel


def _packed(tensors) -> bytes:
    """Their addresses, one machine word each."""
    return array("Q", map(_data_ptr, tensors)).tobytes()


def _addresses(grads: List[Optional[torch.Tensor]], dtype: torch.dtype) -> Optional[bytes]:
    """``_packed(grads)``; None unless every gradient is there, contiguous and of ``dtype``."""
    if _native is not None:
        return _native.tensor_addresses(grads, dtype)
    for g in grads:
        if g is None or g.dtype != dtype or g.layout != torch.strided or not g.is_contiguous():
            return None
    return _packed(grads)


def _own_step(impl):
    """``step`` as ``torch.optim.Optimizer`` would wrap it, minus the cost: torch puts every optimizer's ``step``
    inside a profiler range and two hook loops (about 10 us per call - a quarter of a whole training step's host
    time on a small model).  Here the registered step hooks are called exactly as torch calls them, the range is
    opened only while a profiler is recording, and gradient mode is switched off without building a context
    object.  The ``hooked`` mark tells ``Optimizer.__init__`` not to wrap the function again."""
    from itertools import chain
    from torch.optim import optimizer as _topt

    def step(self, *args, **kwargs):
        full = (self,) + args
        if _topt._global_optimizer_pre_hooks or self._optimizer_step_pre_hooks:
            for hook in chain(_topt._global_optimizer_pre_hooks.values(), self._optimizer_step_pre_hooks.values()):
                result = hook(self, full, kwargs)
                if result is not None:
                    if isinstance(result, tuple) and len(result) == 2:
                        full, kwargs = result
                    else:
                        raise RuntimeError(f"{hook} must return None or a tuple of (new_args, new_kwargs), but got {result}.")
        grad_was_on = torch.is_grad_enabled()
        if grad_was_on:
            torch._C._set_grad_enabled(False)
        try:
            if torch.autograd._profiler_enabled():
                with torch.autograd.profiler.record_function(f"Optimizer.step#{self.__class__.__name__}.step"):
                    out = impl(*full, **kwargs)
            else:
                out = impl(*full, **kwargs)
        finally:
            if grad_was_on:
                torch._C._set_grad_enabled(True)
        if _topt._global_optimizer_post_hooks or self._optimizer_step_post_hooks:
            for hook in chain(self._optimizer_step_post_hooks.values(), _topt._global_optimizer_post_hooks.values()):
                hook(self, full, kwargs)
        return out

    step.hooked = True
    step.__doc__ = impl.__doc__
    step.__wrapped__ = impl
    return step


class _Steady:
    """What a group's last full step established, for the steps after it: as long as the same parameters all
    have contiguous gradients of the same dtype, a step is one pointer comparison per gradient and one launch."""
    __slots__ = ("params", "n", "param_ids", "table", "key", "grad_ptrs", "grad_dtype", "steps_buf", "steps_np", "count", "device",
                 "param_ptr_ends", "fed_by", "numels")

    def same(self, params: List[torch.Tensor]) -> bool:
        """Whether ``params``, which has their number, holds the record's very parameters."""
        if type(self.params) is not tuple:
            return self.params.holds(params)
        return all(map(is_, self.params, params))

    def addresses(self, grads: List[Optional[torch.Tensor]]) -> Optional[bytes]:
        """Where the parameters' gradients lie; None unless each parameter has one that the table can read, that is also of
        the size the table was made for."""
        if type(self.params) is not tuple:
            return self.params.addresses_of(grads, self.grad_dtype)
        if any(g is not None and (g.numel() != n or g.device != self.device) for g, n in zip(grads, self.numels)):
            return None
        return _addresses(grads, self.grad_dtype)


class _FusedBase(torch.optim.Optimizer):
    #: what a copy (``copy.deepcopy``, pickle) takes along beside torch's own; gate, gradient sources and model copies are
    #: addresses of the original's surroundings and stay behind
    _copied: Tuple[str, ...] = ()

    def __init__(self, params, defaults):
        super().__init__(params, defaults)
        self._begin()

    def __getstate__(self) -> Dict:
        return {**super().__getstate__(), **{name: self.__dict__[name] for name in self._copied}}

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        if "_steady" not in self.__dict__:      # a copy (``load_state_dict`` comes here too)
            self._begin()

    def _begin(self) -> None:
        self._steady: Dict[int, _Steady] = {}
        self._tables: Dict[Tuple, Tuple[_lib.OptimTable, Tuple, List]] = {}
        self._model_copies: Dict[int, torch.Tensor] = {}
        self._steps: Dict[int, Tuple[torch.Tensor, int]] = {}     # id(param) -> (its step tensor, value)
        #: device pointer of an ``rg_step_result`` (``TensorPlan.plan.result_device_ptr()``): the step
        #: multiplies the gradients by its clip coefficient and does nothing when it says "skipped".
        #: The host-side bookkeeping (step counts, the first-step flag of momentum buffers) advances
        #: regardless, so a caller that sets ``gate`` must itself skip ``step()`` whenever the device
        #: would (``amp`` does: a dynamic scaler skips on the host, a static one never gates).
        self.gate: int = 0
        #: every gradient is multiplied by this first
        self.grad_scale: float = 1.0
        #: device address of a float to multiply by instead (a loss scaler's ``1 / scale`` kept on the device,
        #: ``rg_scaler_state.inv_scale``), so that a step recorded in a HIP graph follows the scale; 0: off
        self.grad_scale_ptr: int = 0
        self._grad_sources: Dict[int, torch.Tensor] = {}
        self._feed = None                          # see set_grad_feed
        self._feed_params: List[torch.Tensor] = []
        self._feed_offsets: Optional[Dict[int, int]] = None
        self._native_lists: Dict[int, "_native.TensorList"] = {}     # group index -> its parameters in the compiled module

    #: the step can read gradients from tensors other than ``param.grad`` (see ``set_grad_sources``)
    reads_grad_sources = True

    def set_grad_sources(self, params, grads) -> None:
        """For the next steps ``grads[i]`` (any supported dtype, e.g. the still-scaled fp16 model
        gradient) is read as the gradient of ``params[i]`` instead of ``params[i].grad``; together
        with ``grad_scale`` and ``gate`` this folds unscale and clip into the step.  Empty lists
        switch it off."""
        self._grad_sources = {id(p): g for p, g in zip(params, grads) if g is not None}
        self._feed, self._feed_params, self._feed_offsets = None, [], None

    def set_grad_feed(self, feed, params) -> None:
        """``set_grad_sources`` for gradients that a table of the compiled module (a ``GradPlan``) holds:
        ``params[i]`` reads the plan's i-th gradient.  A group whose parameters are a run of ``params`` and whose
        last step left a steady-state record gets the new addresses pushed into its table by the compiled module -
        no Python loop over the parameters; anything else falls back to the tensors themselves."""
        self._grad_sources = {}
        self._feed, self._feed_params = feed, params
        offsets: Optional[Dict[int, int]] = {}
        off = 0
        for gi, group in enumerate(self.param_groups):
            ps = group["params"]
            n = len(ps)
            if n == 0:
                continue
            if off + n > len(params) or ps[0] is not params[off] or ps[-1] is not params[off + n - 1]:
                offsets = None
                break
            offsets[gi] = off
            off += n
        self._feed_offsets = offsets

    def _sources_from_feed(self) -> None:
        """The fed gradients as tensors, for the paths that look at every parameter."""
        if self._feed is not None and not self._grad_sources:
            self._grad_sources = {id(p): g for p, g in zip(self._feed_params, self._feed.sources()) if g is not None}

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        for st in self.state.values():          # a checkpoint may hold moments in another memory order (channels last)
            for name, value in st.items():
                if torch.is_tensor(value) and value.layout == torch.strided and not value.is_contiguous():
                    st[name] = value.contiguous()
        self._steady.clear()          # the state tensors are new objects: the next step rebuilds tables and counters
        self._tables.clear()
        self._steps.clear()

    def invalidate_tables(self) -> None:
        """Forget what earlier steps established about where parameters, gradients, state and model copies live.
        For code that re-homes a parameter's ``.data`` (or a model copy) between steps: the next step then looks at
        every tensor again and pushes all addresses to the device."""
        self._steady.clear()
        self._tables.clear()
        self._native_lists.clear()

    def _steady_grads(self, gi: int, group) -> Optional["_Steady"]:
        """The group's steady-state record, its table pointing at this step's gradients, or None when anything about
        the group differs from the step that made the record (then the full path runs and makes a new one)."""
        st = self._steady.get(gi)
        params = group["params"]
        if st is None or len(params) != st.n:
            return None
        if self._feed is not None and not self._grad_sources:
            off = self._feed_offsets.get(gi) if self._feed_offsets is not None else None
            # (a feed is the compiled module's, and so is the record's list then)
            if (off is not None and st.params.rows_of(params, self._feed_params, off) and self._feed.held() >= off + st.n
                    and dtype_code(st.grad_dtype) == self._feed.source_dtype() and (params[0].data_ptr(), params[-1].data_ptr()) == st.param_ptr_ends):
                if st.fed_by is not self._feed:
                    self._feed.forget_optim(st.table.handle)      # whatever an earlier table at this address was told
                    st.fed_by = self._feed
                if self._feed.push_sources_to_optim(st.table.handle, off, st.n) or st.grad_ptrs is not None:
                    # the table was re-pointed behind the back of the records kept here: they no longer say where it
                    # points, so that a later step through the general path pushes every address again
                    st.grad_ptrs = None
                    hit = self._tables.get(st.key)
                    if hit is not None and hit[0] is st.table:
                        self._tables[st.key] = (hit[0], None, hit[2])
                return st
            self._sources_from_feed()
        # a parameter whose storage was replaced (``p.data = ...``) since the record was made: first and last are
        # looked at here, code that re-homes others calls ``invalidate_tables``
        if (params[0].data_ptr(), params[-1].data_ptr()) != st.param_ptr_ends:
            return None
        if not self._grad_sources and type(st.params) is not tuple:
            found = st.params.grad_addresses_in(params, st.grad_dtype)
        elif not st.same(params):
            return None
        elif self._grad_sources:
            found = st.addresses(list(map(self._grad_sources.get, st.param_ids)))
        else:
            found = st.addresses([p.grad for p in params])
        if found is None:
            return None
        if found != st.grad_ptrs:
            ptrs = list(memoryview(found).cast("Q"))
            st.table.update_pointers(grads=ptrs, stream=stream_handle(st.device))
            st.grad_ptrs = found
            st.fed_by = None      # a feed's record of what it last pushed into this table is stale from here on
            # the full path's record of what the table points at must not outlive this re-pointing: a later
            # full step with the old addresses would otherwise find them "unchanged" and skip the update
            hit = self._tables.get(st.key)
            if hit is not None and hit[0] is st.table and hit[1] is not None:
                self._tables[st.key] = (hit[0], (hit[1][0], tuple(ptrs)) + tuple(hit[1][2:]), hit[2])
        return st

    def _make_steady(self, gi: int, group, table, grads: List[torch.Tensor], count: Optional[int]) -> None:
        params = group["params"]
        st = _Steady()
        st.params, st.n = _native.TensorList(params) if _native is not None else tuple(params), len(params)
        st.numels = table.cache_key[-1]
        st.param_ids = [id(p) for p in params]
        st.table = table
        st.key = table.cache_key
        st.param_ptr_ends = (params[0].data_ptr(), params[-1].data_ptr())
        st.grad_ptrs = _packed(grads)
        st.fed_by = None
        st.grad_dtype = grads[0].dtype
        st.device = params[0].device
        st.count = count
        st.steps_buf = st.steps_np = None
        if count is not None:
            # every parameter's ``step`` becomes a view of one host vector: a step is one add, not one per parameter
            st.steps_buf = torch.full((len(params),), float(count), dtype=torch.float32)
            st.steps_np = st.steps_buf.numpy()          # same memory; numpy adds to a short vector in a tenth of the time
            for i, p in enumerate(params):
                self.state[p]["step"] = st.steps_buf[i]
                self._steps.pop(id(p), None)      # from here on the tensor itself is the count
        self._steady[gi] = st

    def zero_grad(self, set_to_none: bool = True) -> None:
        """``torch.optim.Optimizer.zero_grad`` without its per-parameter bookkeeping."""
        if not set_to_none:
            return super().zero_grad(set_to_none=False)
        for gi, group in enumerate(self.param_groups):
            params = group["params"]
            if _native is None:
                for p in params:
                    p.grad = None
                continue
            # a list may be given other entries in place, so every one is compared (about 1 ns each)
            known = self._native_lists.get(gi)
            if known is None or not known.clear_grads_in(params):
                known = self._native_lists[gi] = _native.TensorList(params)
                known.clear_grads()

    def _scale_source(self, table: _lib.OptimTable) -> _lib.OptimTable:
        """Tell the table where the gradient scale lives, when that changed since its last launch."""
        if getattr(table, "scale_source", 0) != self.grad_scale_ptr:
            table.set_grad_scale_source(self.grad_scale_ptr)
            table.scale_source = self.grad_scale_ptr
        return table

    def _grad_of(self, p: torch.Tensor) -> Optional[torch.Tensor]:
        if self._feed is not None:
            self._sources_from_feed()
        return self._grad_sources.get(id(p), p.grad) if self._grad_sources else p.grad

    # -- model copies (amp): written by the step kernel instead of a separate copy pass
    writes_model_copies = True

    def set_model_copies(self, masters, models) -> None:
        """``models[i]`` (fp16/bf16/fp32, same size) receives ``round(masters[i])`` at every step."""
        for m, c in zip(masters, models):
            if c.numel() != m.numel() or not c.is_contiguous() or c.device != m.device:
                raise ValueError("model copy must be a contiguous tensor of the master's size and device")
            dtype_code(c.dtype)
            self._model_copies[id(m)] = c
        self.invalidate_tables()

    def _check_param(self, p: torch.Tensor, g: torch.Tensor) -> None:
        if p.dtype != torch.float32:
            raise ValueError(f"fused optimizers step fp32 parameters (masters), got {p.dtype}")
        if not p.is_cuda or not p.is_contiguous():
            raise ValueError("fused optimizers need contiguous GPU parameters")
        if g.is_sparse:
            raise ValueError("sparse gradients are not supported")
        if not g.is_contiguous() or g.device != p.device or g.numel() != p.numel():
            raise ValueError("gradient must be contiguous, on the parameter's device and of its size")
        if g.dtype not in _CODES:
            dtype_code(g.dtype)

    @staticmethod
    def _check_rows(params, copies, state1, state2, scales) -> None:
        """What a table is pointed at beside the gradients has to fit the parameters as they are now: a table knows addresses
        and the parameters' sizes only."""
        dtype = torch.float32 if scales is None else torch.float8_e4m3fn
        for i, p in enumerate(params):
            if p.device != params[0].device:
                raise ValueError("the parameters of a group must be on one device")
            held = [(column[i], dtype, p.numel()) for column in (state1, state2) if column is not None]
            if scales is not None:
                held += [(column[i], torch.float32, _lib.state8_num_scales(p.numel())) for column in scales]
            if copies[i] is not None:
                held.append((copies[i], copies[i].dtype, p.numel()))
            for t, want, numel in held:
                if t.dtype != want or t.numel() != numel or t.device != p.device or not t.is_contiguous():
                    raise ValueError(f"parameter {i} has {p.numel()} elements on {p.device}; of its state or model copy, a tensor has "
                                     f"{t.numel()} elements, {t.dtype}, on {t.device}{'' if t.is_contiguous() else ', not contiguous'}")

    def _table(self, key: Tuple, params: List[torch.Tensor], grads: List[torch.Tensor],
               state1: Optional[List[torch.Tensor]], state2: Optional[List[torch.Tensor]],
               scales: Optional[Tuple[List[torch.Tensor], List[torch.Tensor]]] = None) -> _lib.OptimTable:
        """Table for this exact list of parameters and gradient dtypes, re-pointed when any address moved.  ``scales``:
        the states are in 8 bits, and these are their blocks' scales."""
        copies = [self._model_copies.get(id(p)) for p in params]
        key = key + (tuple([g.dtype for g in grads]), tuple(map(_numel, params)))      # what a table cannot change
        def addresses(tensors):
            return tuple(map(_data_ptr, tensors)) if tensors is not None else None
        ptrs = (addresses(params), addresses(grads), addresses(state1), addresses(state2),
                tuple([c.data_ptr() if c is not None else 0 for c in copies]))
        scale_ptrs = tuple(map(addresses, scales)) if scales is not None else (None, None)
        ptrs += scale_ptrs
        hit = self._tables.get(key)
        dev = params[0].device
        if hit is not None and scales is not None and hit[2][4] != (ptrs[2], ptrs[3]) + scale_ptrs:
            hit = None          # 8-bit states have moved, which a table cannot follow: make another
        if hit is None or hit[1] != ptrs:
            self._check_rows(params, copies, state1, state2, scales)
        if hit is None:
            table = _lib.OptimTable(dev.index, ptrs[0], ptrs[1], ptrs[2], ptrs[3],
                                    ptrs[4] if any(ptrs[4]) else None, [p.numel() for p in params],
                                    [dtype_code(g.dtype) for g in grads],
                                    [dtype_code(c.dtype) if c is not None else _lib.RG_F32 for c in copies], *scale_ptrs)
        else:
            table, old, _ = hit
            if old != ptrs:
                state_ptrs = (ptrs[2], ptrs[3]) if scales is None else (None, None)
                table.update_pointers(ptrs[0], ptrs[1], *state_ptrs, ptrs[4] if any(ptrs[4]) else None, stream_handle(dev))
        # the table borrows raw pointers: keep what it points at alive - except the gradients, which only have to
        # live until the launch that reads them is queued (their memory is reused in stream order) and whose
        # release lets the next backward find the same addresses free
        self._tables[key] = (table, ptrs, [params, state1, state2, copies, (ptrs[2], ptrs[3]) + scale_ptrs, scales])
        table.cache_key = key
        return table


class FusedAdam(_FusedBase):
    """``torch.optim.Adam`` (amsgrad off) as one launch per parameter group."""

    _decoupled = False
    _copied = ("capturable", "state_bits", "_buffers8")

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, maximize=False,
                 capturable=False, state_bits=32):
        """``state_bits=8``: both moments are held in 8 bits (``ranncgrad.h``, "optimizer states in 8 bits"): a byte an
        element and a float32 scale for every 256 of them, a quarter of the moments' memory and traffic.  exp_avg_sq is
        held as its root, and a step rounds with a dither that depends on the step count and the element's place alone,
        so that a run can be repeated bit for bit.  Over a run exp_avg_sq comes out 4-8 % too large and single roots 15-20 % (rms)
        off the float32 ones; the same gradients move parameters as with 32 bits but for about 1 % in length and an angle of 4
        degrees (2,000 steps).  ``state[p]`` then has the codes under ``exp_avg`` / ``exp_avg_sq``
        and the scales under ``exp_avg_scale`` / ``exp_avg_sq_scale``; ``state_dict()`` gives, and ``load_state_dict()``
        takes, the float32 moments of ``torch.optim.Adam`` - converted on the GPU, which holds both forms meanwhile.  What
        ``state_dict()`` gave loads back as the same codes and scales (but for about one block in two million, see
        ``rg_state8_quantize``).  Everything else works as with 32 bits.

        ``capturable``: as in ``torch.optim.Adam`` - the step count lives on the device (``state["step"]`` is a
        0-dim float32 GPU tensor), nothing about a step is decided on the host, and ``step()`` may be recorded in
        a HIP graph and replayed.  Every parameter of a group must then have a gradient at every step, at the same
        address (graph capture needs that anyway), and the first ``step()`` - which allocates the state - has to
        run outside a capture.

        What a capture freezes: ``lr``, ``betas``, ``eps``, ``weight_decay`` and ``maximize`` of every group, and
        ``grad_scale`` when it is passed by value, are kernel arguments and so become part of the recorded graph -
        changing ``param_groups[i]["lr"]`` afterwards affects eager steps only, a replayed graph keeps the values
        of the capture (record a new graph after a learning-rate change, and after ``load_state_dict``, which makes new state
        tensors).  What a replay does follow, because it
        is read from device memory: the step count and its bias corrections, the gate (clip coefficient, skip)
        and, with ``grad_scale_ptr``, 1 / loss scale."""
        if lr < 0 or eps < 0 or not 0 <= betas[0] < 1 or not 0 <= betas[1] < 1 or weight_decay < 0:
            raise ValueError("invalid Adam hyper-parameters")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits!r}")
        self.capturable = bool(capturable)
        self.state_bits = int(state_bits)
        self._buffers8: Dict[int, List[Dict[str, torch.Tensor]]] = {}      # group index -> the buffers its 8-bit states lie in
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize))

    def _begin(self) -> None:
        super()._begin()
        if self.state_bits == 8:
            self._conversion_hook = super().register_state_dict_post_hook(FusedAdam._give_moments)
        self._clocks: Dict[int, torch.Tensor] = {}       # group index -> its rg_adam_clock (8 float32 words on the device)

    def _make_moments(self, gi: int, params: List[torch.Tensor], loaded: Optional[List[Dict]] = None) -> None:
        """Moments for ``params`` of one group: zeros (with a count of zero where there is none), or in 8 bits what ``loaded``
        holds in 32.  All of them or, when something raises, none."""
        if not params:
            return
        if self.state_bits == 32:
            made = [{name: torch.zeros_like(p, memory_format=torch.preserve_format) for name in ("exp_avg", "exp_avg_sq")}
                    for p in params]
            self._add_state(params, made)
            return
        buffers: Dict[str, torch.Tensor] = {}
        made = [{} for _ in params]
        for name in ("exp_avg", "exp_avg_sq"):
            codes, scales, buffers[name], buffers[name + "_scale"] = allocate_state8(params)
            for entry, c, s in zip(made, codes, scales):
                entry[name], entry[name + "_scale"] = c, s
        if loaded is not None:
            self._convert_moments(made, loaded, to_codes=True)
        self._add_state(params, made)
        self._buffers8.setdefault(gi, []).append(buffers)

    def _add_state(self, params: List[torch.Tensor], made: List[Dict[str, torch.Tensor]]) -> None:
        steps = [self.state[p]["step"] if "step" in self.state.get(p, {}) else torch.tensor(0.0, dtype=torch.float32) for p in params]
        for p, step, entry in zip(params, steps, made):
            self.state[p].update(step=step, **entry)

    def _moments(self, params: List[torch.Tensor]):
        """The state columns ``_table`` takes for these parameters."""
        def column(name):
            return [self.state[p][name] for p in params]
        if self.state_bits == 32:
            return column("exp_avg"), column("exp_avg_sq")
        return column("exp_avg"), column("exp_avg_sq"), (column("exp_avg_scale"), column("exp_avg_sq_scale"))

    def state_buffers(self, group: int = 0) -> Dict[str, torch.Tensor]:
        """The flat buffers that hold a group's 8-bit states: ``exp_avg`` and ``exp_avg_sq`` (the codes, each parameter's at
        a multiple of 256, in the group's order) and ``exp_avg_scale`` and ``exp_avg_sq_scale`` (a float for every 256)."""
        if self.state_bits != 8:
            raise RuntimeError("state_buffers: the states are in 32 bits, one tensor each")
        held = self._buffers8.get(group, [])
        if len(held) != 1:
            raise RuntimeError("state_buffers: the group's states are not there yet" if not held else
                               "state_buffers: the group's states came in more than one step and lie in several buffers")
        ends = {name: (b.data_ptr(), b.data_ptr() + b.numel() * b.element_size()) for name, b in held[0].items()}
        for p in self.param_groups[group]["params"]:
            st = self.state.get(p, {})
            for name, (first, last) in ends.items():
                if name in st and st[name].numel() and not first <= st[name].data_ptr() < last:
                    raise RuntimeError(f"state_buffers: a parameter's {name} has been given memory of its own")
        return dict(held[0])

    @staticmethod
    def _convert_moments(held: List[Dict], entries: List[Dict], to_codes: bool) -> None:
        """Between the 8-bit states in ``held`` and the float32 moments in ``entries``."""
        by_device: Dict[torch.device, List[int]] = {}
        for i, st in enumerate(held):
            by_device.setdefault(st["exp_avg"].device, []).append(i)
        for rows in by_device.values():
            values, codes, scales, roots = [], [], [], []
            for name in ("exp_avg", "exp_avg_sq"):
                values += [entries[i][name] for i in rows]
                codes += [held[i][name] for i in rows]
                scales += [held[i][name + "_scale"] for i in rows]
                roots += [name == "exp_avg_sq"] * len(rows)
            plan = State8Plan(values, codes, scales, roots)
            if to_codes:
                plan.quantize()
            else:
                plan.dequantize()
            plan.close()

    def register_state_dict_post_hook(self, hook, prepend: bool = False):
        handle = super().register_state_dict_post_hook(hook, prepend)
        if self.state_bits == 8:        # the conversion stays the first of them: hooks see float32 moments
            self._optimizer_state_dict_post_hooks.move_to_end(self._conversion_hook.id, last=False)
        return handle

    def _give_moments(self, packed: Dict) -> Dict:
        """The 8-bit states of what ``state_dict`` has packed as float32 moments."""
        # the packed entries are the live ones of ``self.state``: the float32 moments go into copies, and so does the step
        # count, lest a later step made one of the two older than the other
        params = [p for group in self.param_groups for p in group["params"]]
        held = [(i, p) for i, p in enumerate(params) if "exp_avg_scale" in packed["state"].get(i, {})]
        entries = []
        for i, p in held:
            entry = {k: v.clone() if torch.is_tensor(v) else v for k, v in packed["state"][i].items() if not k.startswith("exp_avg")}
            for name in ("exp_avg", "exp_avg_sq"):        # on the GPU, also where the parameter has gone to the host
                entry[name] = torch.empty(p.shape, dtype=torch.float32, device=self.state[p][name].device)
            entries.append(entry)
        self._convert_moments([self.state[p] for _, p in held], entries, to_codes=False)
        packed["state"] = dict(packed["state"])
        packed["state"].update((i, entry) for (i, _), entry in zip(held, entries))
        return packed

    def load_state_dict(self, state_dict) -> None:
        if any("exp_avg_scale" in st for st in state_dict.get("state", {}).values()):
            raise ValueError("the state dict holds 8-bit codes and scales; states are loaded from the float32 moments that "
                             "state_dict() gives")
        super().load_state_dict(state_dict)
        self._clocks.clear()          # re-seeded from the loaded ``step`` values by the next step
        if self.state_bits == 32:
            return
        self._buffers8.clear()
        for gi, group in enumerate(self.param_groups):
            if all(p.is_cuda for p in group["params"]):       # otherwise they are converted by the step that needs them
                self._settle_moments(gi, group["params"])

    def _settle_moments(self, gi: int, params: List[torch.Tensor]) -> None:
        """Loaded float32 moments among the states of ``params`` into 8 bits."""
        if self.state_bits == 32:
            return
        loaded = [p for p in params if p.is_cuda and "exp_avg" in self.state.get(p, {}) and "exp_avg_scale" not in self.state[p]]
        if not loaded:
            return
        entries = []
        for p in loaded:
            st = self.state[p]
            if st["exp_avg"].numel() != p.numel() or st["exp_avg_sq"].numel() != p.numel():
                raise ValueError("loaded moments differ in size from their parameter")
            entries.append({k: st[k].to(p.device, torch.float32).contiguous() for k in ("exp_avg", "exp_avg_sq")})
        self._make_moments(gi, loaded, entries)

    def _capturable_step(self, gi: int, group) -> None:
        """One group's step with its count on the device: advance the clock (one thread), then the update kernel."""
        params = group["params"]
        if not params:
            return
        # the clock's kernel would have counted the step by the time the update is refused for these
        if not (group["eps"] >= 0 and group["weight_decay"] >= 0):
            raise ValueError(f"invalid Adam hyper-parameters: eps {group['eps']}, weight_decay {group['weight_decay']}")
        clock = self._clocks.get(gi)
        st = self._steady_grads(gi, group) if clock is not None else None
        if st is not None:
            # same parameters, all with usable gradients, as at the step that made the record: the table is in place
            # (re-pointed at the gradients by _steady_grads), only the two launches remain
            b1, b2 = group["betas"]
            stream = stream_handle(st.device)
            _lib.adam_clock_advance(clock.data_ptr(), group["lr"], b1, b2, self.gate, st.device.index, stream)
            self._scale_source(st.table).adam_step_clocked(clock.data_ptr(), group["lr"], b1, b2, group["eps"],
                                                           group["weight_decay"], decoupled=self._decoupled,
                                                           maximize=group["maximize"], grad_scale=self.grad_scale,
                                                           gate=self.gate, stream=stream)
            return
        self._steady.pop(gi, None)
        grads = [self._grad_of(p) for p in params]
        if any(g is None for g in grads):
            raise RuntimeError("a capturable optimizer needs a gradient for every parameter at every step")
        dev = params[0].device
        for p, g in zip(params, grads):
            self._check_param(p, g)
        fresh = [p for p in params if "exp_avg" not in self.state.get(p, {})]
        if clock is None:
            counts = {0 if "exp_avg" not in self.state.get(p, {}) else int(self.state[p]["step"]) for p in params}
            if len(counts) != 1:
                raise RuntimeError("a capturable optimizer keeps one step count per group; the loaded counts differ")
        elif fresh:
            raise RuntimeError("a capturable optimizer keeps one step count per group: a parameter without moments joined it")
        self._make_moments(gi, fresh)
        self._settle_moments(gi, params)
        table = self._table((gi, "capturable", tuple(id(p) for p in params)), list(params), grads, *self._moments(params))
        if clock is None:
            clock = torch.zeros(_lib.ADAM_CLOCK_BYTES // 4, dtype=torch.float32, device=dev)
            count = counts.pop()
            if count:
                clock.view(torch.int64)[0] = count
                clock[4] = float(count)
            for p in params:
                self.state[p]["step"] = clock[4]          # every parameter's count is the group's, on the device
            self._clocks[gi] = clock
        b1, b2 = group["betas"]
        stream = stream_handle(dev)
        _lib.adam_clock_advance(clock.data_ptr(), group["lr"], b1, b2, self.gate, dev.index, stream)
        self._scale_source(table).adam_step_clocked(clock.data_ptr(), group["lr"], b1, b2, group["eps"], group["weight_decay"],
                                decoupled=self._decoupled, maximize=group["maximize"], grad_scale=self.grad_scale,
                                gate=self.gate, stream=stream)
        self._make_steady(gi, group, table, grads, None)

    @_own_step
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self.capturable:
            for gi, group in enumerate(self.param_groups):
                self._capturable_step(gi, group)
            return loss
        for gi, group in enumerate(self.param_groups):
            st = self._steady_grads(gi, group)
            if st is not None:
                b1, b2 = group["betas"]
                self._scale_source(st.table).adam_step(group["lr"], b1, b2, group["eps"], group["weight_decay"], st.count + 1,
                                   decoupled=self._decoupled, maximize=group["maximize"], grad_scale=self.grad_scale,
                                   gate=self.gate, stream=stream_handle(st.device))
                st.count += 1                    # behind the launch: a step that is refused does not count
                st.steps_np += 1.0
                continue
            self._steady.pop(gi, None)
            by_step: Dict[int, Tuple[List[torch.Tensor], List[torch.Tensor]]] = {}       # count -> parameters, their counts
            grad_of: Dict[int, torch.Tensor] = {}
            found = []
            for p in group["params"]:            # everything that can be refused or fail comes before the first launch,
                g = self._grad_of(p)
                if g is None:
                    continue
                self._check_param(p, g)
                found.append(p)
                grad_of[id(p)] = g
            held = [self.state.get(p) for p in found]         # (a tensor's hash is a call into Python: looked up once)
            fresh = [p for p, st in zip(found, held) if st is None or "exp_avg" not in st]
            self._make_moments(gi, fresh)
            self._settle_moments(gi, group["params"])
            if fresh:
                held = [self.state[p] for p in found]
            for p, st in zip(found, held):
                # ``step`` stays a tensor (torch.optim's state layout); its integer value is mirrored
                # here so that a step costs one batched increment instead of one tensor op per parameter
                t = st["step"]
                if not isinstance(t, torch.Tensor):
                    t = st["step"] = torch.tensor(float(t), dtype=torch.float32)
                seen = self._steps.get(id(p))
                ps, counts = by_step.setdefault((seen[1] if seen is not None and seen[0] is t else int(t)) + 1, ([], []))
                ps.append(p)
                counts.append(t)
            tables = [self._table((gi, tuple(map(id, ps))), ps, [grad_of[id(p)] for p in ps], *self._moments(ps))
                      for ps, _ in by_step.values()]
            for table, (step, (ps, counts)) in zip(tables, by_step.items()):
                b1, b2 = group["betas"]
                self._scale_source(table).adam_step(group["lr"], b1, b2, group["eps"], group["weight_decay"], step,
                                decoupled=self._decoupled, maximize=group["maximize"], grad_scale=self.grad_scale,
                                gate=self.gate, stream=stream_handle(ps[0].device))
                torch._foreach_add_(counts, 1)                        # ... and the counts move behind it
                for p, t in zip(ps, counts):
                    self._steps[id(p)] = (t, step)
                if len(by_step) == 1 and len(ps) == len(group["params"]):
                    self._make_steady(gi, group, table, [grad_of[id(p)] for p in ps], step)
        return loss


class FusedAdamW(FusedAdam):
    """``torch.optim.AdamW``: weight decay applied to the parameter, not the gradient."""

    _decoupled = True

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, maximize=False,
                 capturable=False, state_bits=32):
        super().__init__(params, lr, betas, eps, weight_decay, maximize, capturable, state_bits)


class FusedSGD(_FusedBase):
    """``torch.optim.SGD`` as one launch per parameter group (two on the step that creates
    momentum buffers for only some of the parameters)."""

    def __init__(self, params, lr=1e-3, momentum=0.0, dampening=0.0, weight_decay=0.0, nesterov=False, maximize=False):
        if lr < 0 or momentum < 0 or weight_decay < 0:
            raise ValueError("invalid SGD hyper-parameters")
        if nesterov and (momentum <= 0 or dampening != 0):
            raise ValueError("Nesterov momentum requires a momentum and zero dampening")
        super().__init__(params, dict(lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay,
                                      nesterov=nesterov, maximize=maximize))

    @_own_step
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            st = self._steady_grads(gi, group)
            if st is not None:
                self._scale_source(st.table).sgd_step(group["lr"], group["momentum"], group["dampening"], group["weight_decay"],
                                  group["nesterov"], group["maximize"], first_step=False, grad_scale=self.grad_scale,
                                  gate=self.gate, stream=stream_handle(st.device))
                continue
            self._steady.pop(gi, None)
            fresh, seasoned, unnamed = [], [], []
            buffer_of: Dict[int, torch.Tensor] = {}
            grad_of: Dict[int, torch.Tensor] = {}
            for p in group["params"]:
                g = self._grad_of(p)
                if g is None:
                    continue
                self._check_param(p, g)
                grad_of[id(p)] = g
                st = self.state.get(p)
                buffer = st.get("momentum_buffer") if st is not None else None
                if group["momentum"] != 0 and buffer is None:
                    # zeros, not empty: if the first launch is gated off on the device the buffer must
                    # not reach the next step with whatever the memory held
                    buffer = torch.zeros_like(p, memory_format=torch.preserve_format)
                    fresh.append(p)
                else:
                    seasoned.append(p)
                    if st is None:
                        unnamed.append(p)
                buffer_of[id(p)] = buffer
            tables = []                          # all of them before the first launch: what fails leaves the state as it was
            for first, ps in ((True, fresh), (False, seasoned)):
                if not ps:
                    continue
                bufs = [buffer_of[id(p)] for p in ps] if group["momentum"] != 0 else None
                tables.append((first, ps, self._table((gi, first, tuple(map(id, ps))), ps, [grad_of[id(p)] for p in ps], bufs, None)))
            for first, ps, table in tables:
                self._scale_source(table).sgd_step(group["lr"], group["momentum"], group["dampening"], group["weight_decay"],
                               group["nesterov"], group["maximize"], first_step=first, grad_scale=self.grad_scale,
                               gate=self.gate, stream=stream_handle(ps[0].device))
                if first:                        # a buffer is the state's once its first step has been launched
                    for p in ps:
                        self.state[p]["momentum_buffer"] = buffer_of[id(p)]
                else:
                    for p in unnamed:            # without momentum a stepped parameter has an empty entry, as in torch.optim
                        self.state[p]
                if not first and not fresh and len(ps) == len(group["params"]):
                    self._make_steady(gi, group, table, [grad_of[id(p)] for p in ps], None)
        return loss
