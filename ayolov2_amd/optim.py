"""``SGD``: torch.optim.SGD's interface and arithmetic with the whole step in ONE HIP launch (``ayolo_sgd_step``).

The reference builds ``optim.SGD(pg_bn, lr, momentum, nesterov=True)`` plus a weight-decay group and a bias group
(scripts/train/yolo_trainer.py:149-168) and steps it through ``torch.cuda.amp.GradScaler``
(yolo_trainer.py:332-338).  This class keeps that surface -- param groups, ``state_dict`` with ``momentum_buffer``
entries, LR schedulers, ``GradScaler.step`` (``_step_supports_amp_scaling``: the scaler hands over ``grad_scale`` and
``found_inf`` tensors and the kernel divides / skips on the device, no host sync) -- but the ~180 parameter tensors are
updated by a single kernel instead of several torch launches per parameter group.  CPU parameters fall back to
torch's own arithmetic (the class is then a plain torch.optim.SGD).

``AdamW``, ``adamw_step``: torch.optim.AdamW's step over many tensors at once (``ayolo_adamw_step``), moments in 32 or in 8 bits;
``grad_norm``, ``clip_grads_``, ``clip_grad_norm_``: the 2-norm of all gradients and clipping by it (``ayolo_grad_norm``,
``ayolo_grad_clip``).  These take their tensors as lists and keep nothing between calls, so a captured call replays as it is."""
from __future__ import annotations

import array
import ctypes
import numbers
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _lib

_MAX_GROUPS = 8
_CHUNK = 32768


class _Group(ctypes.Structure):
    _fields_ = [("lr", ctypes.c_float), ("momentum", ctypes.c_float), ("weight_decay", ctypes.c_float),
                ("dampening", ctypes.c_float), ("nesterov", ctypes.c_int), ("reserved", ctypes.c_int)]


class _Groups(ctypes.Structure):
    _fields_ = [("g", _Group * _MAX_GROUPS)]


_JOB = np.dtype([("p", "<u8"), ("g", "<u8"), ("buf", "<u8"), ("n", "<i8"), ("group", "<i4"), ("first", "<i4")])


class SGD(torch.optim.SGD):
    _step_supports_amp_scaling = True

    def __init__(self, params, lr=1e-3, momentum=0.0, dampening=0.0, weight_decay=0.0, nesterov=False):
        super().__init__(params, lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay,
                         nesterov=nesterov)
        self._table = None          # {gradient pointers: built job table}
        self._plist = None

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        self._table = None                  # momentum buffers were replaced

    @staticmethod
    def _dense_like(p: torch.Tensor, g: torch.Tensor) -> torch.Tensor:
        """The gradient in the parameter's own memory order (a no-op for the plan's gradients)."""
        if g.stride() == p.stride():
            return g
        out = torch.empty_like(p)          # preserve_format: same strides as p for dense tensors
        out.copy_(g)
        return out

    def _build_table(self, plist, grads):
        """Validate + lay out the job table (only when a parameter / gradient / momentum pointer changed)."""
        rows, keep, dev = [], [], None
        for (gi, p), g in zip(plist, grads):
            if g is None:
                continue
            if not (p.is_cuda and p.dtype == torch.float32 and g.dtype == torch.float32 and not g.is_sparse):
                return None
            dense = p.is_contiguous() or (p.dim() == 4 and p.is_contiguous(memory_format=torch.channels_last))
            if not dense:
                raise _lib.AyoloError("ayolov2_amd.optim.SGD: parameter is not a dense block of memory")
            dev = p.device
            gr = self._dense_like(p, g)
            if gr is not g:
                keep.append(gr)            # a re-laid-out copy lives as long as the table; the caller's own gradient
                                           # tensors are NOT retained (the key validates their addresses)
            buf = None
            if float(self.param_groups[gi]["momentum"]) != 0.0:
                st = self.state[p]
                buf = st.get("momentum_buffer")
                if buf is None:
                    # NaN = "not initialised yet": the kernel then takes buf = g, and a first step skipped by the
                    # GradScaler (found_inf is only known on the device) leaves the buffer uninitialised, like torch
                    buf = st["momentum_buffer"] = torch.full_like(p, float("nan"))
                elif buf.stride() != p.stride() or not buf.is_cuda:
                    nb = torch.empty_like(p)
                    nb.copy_(buf)
                    buf = st["momentum_buffer"] = nb
            # chunks of <= _CHUNK elements: one grid row each, so the few multi-million-element conv weights are spread
            # over hundreds of workgroups instead of being walked by one row of the grid
            n, pb, gb, bb = p.numel(), p.data_ptr(), gr.data_ptr(), buf.data_ptr() if buf is not None else 0
            for o in range(0, n, _CHUNK):
                rows.append((pb + 4 * o, gb + 4 * o, bb + 4 * o if bb else 0, min(_CHUNK, n - o), gi, 0))
        if not rows:
            return ()
        jobs = np.array(rows, dtype=_JOB)
        # pinned staging + asynchronous copy: a pageable .to(device) would block the host until the stream has drained
        host = torch.from_numpy(jobs.view(np.uint8).copy()).pin_memory()
        tab = host.to(dev, non_blocking=True)
        copied = len(keep) > 0
        keep.append(host)
        return tab, len(rows), keep, copied

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        ngroups = len(self.param_groups)
        sig = tuple(len(g["params"]) for g in self.param_groups)
        if self._plist is None or self._plist[0] != sig:
            self._plist = (sig, [(gi, p) for gi, g in enumerate(self.param_groups) for p in g["params"]])
            self._table = None
        plist = self._plist[1]
        grads = [p.grad for _, p in plist]
        # host cost matters (the train step keeps the host ~1 step ahead of the GPU at best): the table is rebuilt only
        # when a pointer changed -- the plan hands out views of one flat gradient buffer, normally at the same address
        key = tuple(0 if g is None else g.data_ptr() for g in grads) + tuple(p.data_ptr() for _, p in plist)
        if self._table is None:
            self._table = {}
        built = self._table.get(key, False)
        if built is False:
            # (the plan's per-step gradient buffer alternates between a few allocator blocks: keep a table per address set)
            built = None
            if ngroups <= _MAX_GROUPS and not any(g.get("maximize", False) for g in self.param_groups):
                built = self._build_table(plist, grads)
            if len(self._table) >= 4:
                self._table.pop(next(iter(self._table)))
            self._table[key] = built
        if built is None:                                      # CPU / exotic parameters: torch's own arithmetic
            if getattr(self, "grad_scale", None) is not None or getattr(self, "found_inf", None) is not None:
                raise _lib.AyoloError("ayolov2_amd.optim.SGD: GradScaler hand-over needs fp32 parameters on the GPU")
            return super().step()
        if built == ():
            return loss
        tab, n, keep, copied = built
        if copied:                                             # a gradient had to be re-laid-out: its content is per step
            self._table.pop(key, None)
        groups = _Groups()
        for gi, g in enumerate(self.param_groups):
            gg = groups.g[gi]
            gg.lr, gg.momentum, gg.weight_decay = float(g["lr"]), float(g["momentum"]), float(g["weight_decay"])
            gg.dampening, gg.nesterov = float(g["dampening"]), int(bool(g["nesterov"]))
        scale = getattr(self, "grad_scale", None)
        found = getattr(self, "found_inf", None)
        _lib.call("ayolo_sgd_step", tab.data_ptr(), n, ctypes.byref(groups),
                  scale.data_ptr() if scale is not None else None, found.data_ptr() if found is not None else None,
                  torch.cuda.current_stream().cuda_stream)
        _lib.bump_versions(p for (_, p), g in zip(plist, grads) if g is not None)     # written through raw pointers
        return loss


# ---------------------------------------------------------------------------------------- gradient norm and clipping
_TENSOR = np.dtype([("data", "<u8"), ("numel", "<i8"), ("layout", "<u8"), ("dtype", "<i4"), ("device", "<i2"), ("present", "<i2")])
MOMENT_BLOCK = 128          # elements of an 8-bit moment that share an exponent


def _device_of(tensors, what: str) -> Optional[torch.device]:
    for t in tensors:
        if t is not None:
            if not torch.is_tensor(t):
                raise _lib.AyoloError(f"{what}: expected a tensor, got {type(t).__name__}")
            if not t.is_cuda:
                raise _lib.AyoloError(f"{what}: the HIP path needs tensors on the GPU (got {t.device}); there is no CPU fallback")
            return t.device
    return None


def _scalar(t: Optional[torch.Tensor], dev: torch.device, what: str, name: str):
    """The address of one fp32 number on the device (None: a null pointer)."""
    if t is None:
        return None
    if not torch.is_tensor(t) or t.dtype != torch.float32 or t.numel() != 1 or t.device != dev:
        raise _lib.AyoloError(f"{what}: {name} must be one fp32 number on {dev}")
    return t.data_ptr()


def grad_norm(grads: Sequence[Optional[torch.Tensor]], grad_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The 2-norm over all elements of all gradients (fp32, fp16 or bf16; None entries are skipped) as one fp32 number on their
    device, divided by the device scalar `grad_scale` if given.  Summed in fp64 in a fixed order."""
    grads = list(grads)
    dev = _device_of(grads, "grad_norm")
    if dev is None:
        return torch.zeros(())
    return _norm(grads, _lib.tensor_rows(grads, "grad_norm"), dev, grad_scale)


def _norm(grads, rows: bytes, dev: torch.device, grad_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    scale = _scalar(grad_scale, dev, "grad_norm", "grad_scale")
    need = int(_lib.lib().ayolo_grad_norm_workspace(rows, len(grads)))
    ws, norm = torch.empty(need, dtype=torch.uint8, device=dev), torch.empty((), dtype=torch.float32, device=dev)
    try:
        _lib.call_on(dev.index, "ayolo_grad_norm", rows, len(grads), scale, norm.data_ptr(), ws.data_ptr(), need)
    except _lib.AyoloError:
        info = np.frombuffer(rows, dtype=_TENSOR)
        if not ((info["layout"] == 0) & (info["present"] != 0)).any():
            raise
        # an expanded or strided gradient (the call launches nothing then): the norm of its elements in a block
        grads = [g if g is None else g.contiguous() for g in grads]
        return _norm(grads, _lib.tensor_rows(grads, "grad_norm"), dev, grad_scale)
    return norm


def clip_grads_(grads: Sequence[Optional[torch.Tensor]], max_norm: float, norm: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Multiplies every gradient by ``min(1, max_norm / (norm + 1e-6))`` in place and returns the norm (a device scalar; computed
    here unless given).  An infinite norm makes finite gradients zero, a NaN norm makes all of them NaN, as the formula does.
    Gradients must be dense blocks of memory that do not overlap."""
    grads = list(grads)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise _lib.AyoloError(f"clip_grads_: max_norm={max_norm}")
    dev = _device_of(grads, "clip_grads_")
    if dev is None:
        return torch.zeros(()) if norm is None else norm
    rows = _lib.tensor_rows(grads, "clip_grads_")
    if norm is None:
        norm = _norm(grads, rows, dev)
    _lib.call_on(dev.index, "ayolo_grad_clip", rows, len(grads), _scalar(norm, dev, "clip_grads_", "norm"), max_norm)
    _lib.host().bump(grads, grads)
    return norm


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ for the 2-norm: clips the parameters' ``.grad`` in place (two launches per 332 tensors and
    one for their sum; gradients that need no clipping are read once and not written) and returns their norm.  Gradients on the CPU go to
    torch's own function."""
    if float(norm_type) != 2.0:
        raise _lib.AyoloError(f"clip_grad_norm_: norm_type={norm_type}: only the 2-norm has a kernel")
    parameters = [parameters] if torch.is_tensor(parameters) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads or not grads[0].is_cuda:
        return torch.nn.utils.clip_grad_norm_(parameters, max_norm, norm_type, error_if_nonfinite)
    norm = grad_norm(grads)
    if error_if_nonfinite and not bool(torch.isfinite(norm)):
        raise RuntimeError("clip_grad_norm_: the gradients' norm is not finite")
    with torch.no_grad():
        return clip_grads_(grads, max_norm, norm)


# --------------------------------------------------------------------------------------------------------------- AdamW
class Moment8(NamedTuple):
    """A moment in 8 bits: one code per element in the parameter's shape and memory order, one exponent per MOMENT_BLOCK codes in that
    order (codes that are copied into another one no longer fit their exponents)."""
    codes: torch.Tensor
    exps: torch.Tensor


def new_moment8(p: torch.Tensor) -> Moment8:
    """An 8-bit moment of zeros for parameter `p`."""
    return Moment8(torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format),
                   torch.zeros(-(-p.numel() // MOMENT_BLOCK), dtype=torch.uint8, device=p.device))


def unpack_moments(moments: Sequence[Moment8], signed: bool, out: Optional[Sequence[torch.Tensor]] = None) -> Sequence[torch.Tensor]:
    """The fp32 values of 8-bit moments, all in one go.  `signed`: first moments (exp_avg), else second ones (exp_avg_sq)."""
    moments = list(moments)
    if not moments:
        return [] if out is None else out
    dev = _device_of((m[0] for m in moments), "unpack_moments")
    if out is None:
        out = [torch.empty_like(m[0], dtype=torch.float32) for m in moments]
    elif len(out) != len(moments):
        raise _lib.AyoloError(f"unpack_moments: {len(out)} outputs for {len(moments)} moments")
    out = list(out)
    _lib.call_on(dev.index, "ayolo_moment_values", _lib.tensor_rows(moments, "unpack_moments", 0), _lib.tensor_rows(moments, "unpack_moments", 1),
                 _lib.tensor_rows(out, "unpack_moments", -1, out), len(moments), int(bool(signed)))
    return out


def _layouts(tensors) -> np.ndarray:
    """A number per tensor that is equal for equal shapes in equal memory order, 0 for what is no dense block of memory."""
    return np.frombuffer(_lib.tensor_rows(tensors, "memory order"), dtype=_TENSOR)["layout"]


def _moment_like(p: torch.Tensor, m: torch.Tensor) -> torch.Tensor:
    """An fp32 moment in parameter `p`'s memory order."""
    return torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(m)


def _in_order_of(p: torch.Tensor, t: torch.Tensor) -> torch.Tensor:
    """A copy of `t` in parameter `p`'s memory order."""
    return torch.empty_like(p, dtype=t.dtype, device=t.device, memory_format=torch.preserve_format).copy_(t.detach())


def _moment8_like(p: torch.Tensor, m: Moment8, signed: bool) -> Moment8:
    """An 8-bit moment in parameter `p`'s memory order.  The exponents belong to blocks of codes in the codes' OWN order: in another
    one the blocks are others, so the values are taken out and put into codes again."""
    own, want = _layouts([m[0], p])
    if own != 0 and own == want:
        codes = torch.empty_like(p, dtype=torch.uint8, memory_format=torch.preserve_format)
        return Moment8(codes.copy_(m[0]), m[1])
    return _pack_moment(_moment_like(p, unpack_moments([m], signed)[0]), signed)


def _pack_moment(x: torch.Tensor, signed: bool) -> Moment8:
    """Fp32 values (a dense block of memory) in 8 bits, by the format of csrc/adamw.hip: the rounding to nearest of one conversion,
    1/16 of a value at most (a step's own rounding is stochastic because it is repeated; this one is not)."""
    bias, least, top = (14, 1, 0x7F) if signed else (30, 10, 0xFF)
    n = x.numel()
    flat = torch.zeros(-(-n // MOMENT_BLOCK) * MOMENT_BLOCK, device=x.device)
    flat[:n] = x.as_strided((n,), (1,))
    flat = flat.view(-1, MOMENT_BLOCK)
    bits = flat.abs().view(torch.int32)
    finite = bits < 0x7F800000
    e = (torch.where(finite, bits, 0).amax(1) >> 23).clamp(min=least) if n else bits.new_zeros(0)
    power = ((bias - e.long() + 1023) << 52).view(torch.float64)          # 2 ** (bias - e)
    y = (torch.where(finite, flat.abs(), 0.0).double() * power[:, None]).float()
    code = (y.view(torch.int32) + 0x80008) >> 20
    if not signed:
        code = torch.where(bits != 0, code.clamp(min=1), code)            # above zero stays above zero
    code = torch.where(finite, code, torch.where(bits == 0x7F800000, top - 1, top))
    if signed:
        code = torch.where((flat.view(torch.int32) < 0) & (bits <= 0x7F800000), code | 0x80, code)
    codes = torch.empty_like(x, dtype=torch.uint8, memory_format=torch.preserve_format)
    codes.as_strided((n,), (1,)).copy_(code.view(-1)[:n])
    return Moment8(codes, e.to(torch.uint8))


def _per_tensor(v, n: int, what: str):
    """(number, None), or (0, n floats as bytes) where a number per tensor is given."""
    if isinstance(v, numbers.Real):
        return float(v), None
    arr = array.array("f", v if type(v) is list else map(float, v))
    if len(arr) != n:
        raise _lib.AyoloError(f"adamw_step: {len(arr)} values of {what} for {n} tensors")
    return 0.0, arr.tobytes()


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[Optional[torch.Tensor]], exp_avgs: Sequence, exp_avg_sqs: Sequence,
               steps: Sequence[torch.Tensor], *, lr: Union[float, torch.Tensor, Sequence[float]], betas: Tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: Union[float, Sequence[float]] = 1e-2, maximize: bool = False, seed: int = 0,
               total_norm: Optional[torch.Tensor] = None, max_norm: Optional[float] = None, grad_scale: Optional[torch.Tensor] = None,
               found_inf: Optional[torch.Tensor] = None) -> None:
    """One AdamW step (torch.optim.AdamW's arithmetic) over lists of tensors, in place, in a few launches for all of them.

    params / grads: fp32, fp16 or bf16 on one GPU, a gradient of its parameter's type (None: that entry stays as it is); dense
    blocks of memory, states in the parameter's memory order (gradients are laid out like it where they are not); what is written
    shares memory with nothing else of the call.  16-bit parameters are rounded to nearest: what is below half a
    step of theirs is lost, so keep fp32 masters for long training.  exp_avgs / exp_avg_sqs: fp32 tensors, or Moment8 pairs
    (new_moment8), rounded stochastically from `seed`, the step, the entry's place in the list and the element.  steps: one fp32
    number per entry on the device, counted up here.  lr: a number, a number per tensor, or a device scalar (which a captured
    step follows); weight_decay: a number, or a number per tensor.  total_norm with max_norm: gradients are multiplied by
    min(1, max_norm / (total_norm + 1e-6)) on the way.  grad_scale: a device scalar that gradients are divided by; found_inf: a
    device scalar, nothing at all is changed where it is not 0 (torch.amp.GradScaler's pair)."""
    _adamw(params, grads, exp_avgs, exp_avg_sqs, steps, None, lr, betas, eps, weight_decay, maximize, seed, total_norm, max_norm, grad_scale,
           found_inf)


def _adamw(params, grads, exp_avgs, exp_avg_sqs, steps, relay, lr, betas, eps, weight_decay, maximize, seed, total_norm, max_norm, grad_scale,
           found_inf) -> None:
    """adamw_step.  relay(places): puts the moments of these entries into their parameters' memory order, in the lists given here
    (None: they are refused)."""
    params, grads = list(params), list(grads)
    n = len(params)
    for other, name in ((grads, "grads"), (exp_avgs, "exp_avgs"), (exp_avg_sqs, "exp_avg_sqs"), (steps, "steps")):
        if len(other) != n:
            raise _lib.AyoloError(f"adamw_step: {len(other)} {name} for {n} params")
    dev = _device_of(grads, "adamw_step")
    if dev is None:
        return
    if (total_norm is None) != (max_norm is None):
        raise _lib.AyoloError("adamw_step: total_norm and max_norm go together")
    bits8 = isinstance(next((m for m in exp_avgs if m is not None), None), (tuple, list))      # pairs throughout, or tensors
    rows, unlike = _lib.tensor_rows, _lib.host().unlike
    L, H = _lib.AdamWList(), _lib.AdamWHyper()
    # (what is written through raw pointers counts its versions here, where a gradient is given)
    P, G = rows(params, "adamw_step: params", -1, grads), rows(grads, "adamw_step: grads")
    other = [i for i in unlike(G, P) if grads[i].shape == params[i].shape]
    if other:                                      # gradients in another memory order than their parameters
        for i in other:
            grads[i] = _in_order_of(params[i], grads[i])
        G = rows(grads, "adamw_step: grads")
    L.n, L.p, L.g = n, P, G
    first = 0 if bits8 else -1
    M, V = rows(exp_avgs, "adamw_step: exp_avgs", first, grads), rows(exp_avg_sqs, "adamw_step: exp_avg_sqs", first, grads)
    if relay is not None:
        other = [i for i in {*unlike(M, P), *unlike(V, P)} if grads[i] is not None]
        if other:
            relay(other)
            M, V = rows(exp_avgs, "adamw_step: exp_avgs", first), rows(exp_avg_sqs, "adamw_step: exp_avg_sqs", first)
    L.m, L.v = M, V
    if bits8:
        L.me, L.ve = rows(exp_avgs, "adamw_step: exp_avgs", 1, grads), rows(exp_avg_sqs, "adamw_step: exp_avg_sqs", 1, grads)
    L.step = rows(steps, "adamw_step: steps", -1, grads)
    if torch.is_tensor(lr):
        H.lr_dev = _scalar(lr, dev, "adamw_step", "lr")
    else:
        H.lr, L.lr = _per_tensor(lr, n, "lr")
    H.weight_decay, L.weight_decay = _per_tensor(weight_decay, n, "weight_decay")
    H.beta1, H.beta2, H.eps = float(betas[0]), float(betas[1]), float(eps)
    H.grad_scale = _scalar(grad_scale, dev, "adamw_step", "grad_scale")
    H.found_inf = _scalar(found_inf, dev, "adamw_step", "found_inf")
    H.norm = _scalar(total_norm, dev, "adamw_step", "total_norm")
    H.max_norm = 0.0 if max_norm is None else float(max_norm)
    H.maximize, H.seed = int(bool(maximize)), int(seed) & 0xFFFFFFFF
    need = int(_lib.lib().ayolo_adamw_workspace(n))
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _lib.call_on(dev.index, "ayolo_adamw_step", L, H, ws.data_ptr(), need)


class AdamW(torch.optim.AdamW):
    """torch.optim.AdamW's interface and arithmetic with the whole step in a few launches (adamw_step).

    ``state_bits=8`` keeps both moments in one byte per element (``exp_avg`` / ``exp_avg_sq`` hold codes, ``exp_avg_exps`` /
    ``exp_avg_sq_exps`` an exponent per 128): 2 bytes of state per parameter instead of 8, rounded stochastically from `seed`.
    ``max_norm`` clips the gradients' global 2-norm inside the step, without writing them.  ``step`` counts on the device, so
    GradScaler's skipped steps do not count and need no host sync, and a step can be captured (after one eager step, which makes
    the states; a learning rate that changes between replays is given as a device scalar).  32-bit state dicts and
    torch.optim.AdamW's load into each other; an 8-bit state dict also loads into a 32-bit optimiser.  States are brought into their
    parameter's memory order when they are loaded and when it changes (8-bit ones are rounded to nearest once).  CPU parameters fall back
    to torch's own arithmetic (32-bit states)."""
    _step_supports_amp_scaling = True

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, maximize=False, state_bits=32,
                 max_norm: Optional[float] = None, seed: int = 0):
        if state_bits not in (8, 32):
            raise _lib.AyoloError(f"ayolov2_amd.optim.AdamW: state_bits={state_bits}: 8 or 32")
        if max_norm is not None and not float(max_norm) >= 0.0:
            raise _lib.AyoloError(f"ayolov2_amd.optim.AdamW: max_norm={max_norm}")
        self.state_bits, self.max_norm, self.seed = state_bits, max_norm, seed
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize)

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "max_norm": self.max_norm, "seed": self.seed}

    def _new_states(self, todo) -> None:
        """States of parameters that have a gradient for the first time."""
        if torch.cuda.is_current_stream_capturing():
            raise _lib.AyoloError("ayolov2_amd.optim.AdamW: run one step before capturing: a replay would start from new states")
        for p, t in zip(todo, torch.zeros(len(todo), dtype=torch.float32, device=todo[0].device).unbind()):
            st = self.state[p]
            st["step"] = t
            if self.state_bits == 8:
                m, v = new_moment8(p), new_moment8(p)
                st["exp_avg"], st["exp_avg_exps"], st["exp_avg_sq"], st["exp_avg_sq_exps"] = m.codes, m.exps, v.codes, v.exps
            else:
                st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
                st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)

    def _states(self, ps, grads):
        """(exp_avgs, exp_avg_sqs, steps) of a group's parameters; None for those that never had a gradient."""
        get = self.state.get
        sts = [get(p) for p in ps]
        todo = [p for p, g, st in zip(ps, grads, sts) if g is not None and not st]
        if todo:
            self._new_states(todo)
            sts = [get(p) for p in ps]
        none = dict.fromkeys(("exp_avg", "exp_avg_sq", "exp_avg_exps", "exp_avg_sq_exps", "step"))
        sts = [st or none for st in sts]
        if self.state_bits == 8:
            pairs = (lambda name: [None if st is none else (st[name], st[name + "_exps"]) for st in sts])
            return pairs("exp_avg"), pairs("exp_avg_sq"), [st["step"] for st in sts]
        return [st["exp_avg"] for st in sts], [st["exp_avg_sq"] for st in sts], [st["step"] for st in sts]

    def _relay(self, ps, ms, vs, which) -> None:
        """Moments into the memory order that their parameters have now (a weight that was made channels-last after its states)."""
        if torch.cuda.is_current_stream_capturing():
            raise _lib.AyoloError("ayolov2_amd.optim.AdamW: run one step before capturing: a parameter's memory order has changed")
        for i in which:
            p, st = ps[i], self.state[ps[i]]
            for name, signed, of in (("exp_avg", True, ms), ("exp_avg_sq", False, vs)):
                if st[name].shape != p.shape:
                    continue
                if self.state_bits == 8:
                    of[i] = st[name], st[name + "_exps"] = _moment8_like(p, Moment8(*of[i]), signed)
                else:
                    of[i] = st[name] = _in_order_of(p, st[name])

    @torch.no_grad()
    def step(self, closure=None):
        scale, found = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        if not next((p.is_cuda for g in self.param_groups for p in g["params"]), True):
            if self.state_bits == 8 or scale is not None or found is not None:
                raise _lib.AyoloError("ayolov2_amd.optim.AdamW: 8-bit states and the GradScaler hand-over need parameters on the GPU")
            if self.max_norm is not None:
                if closure is not None:
                    raise _lib.AyoloError("ayolov2_amd.optim.AdamW: max_norm with a closure needs parameters on the GPU")
                torch.nn.utils.clip_grad_norm_([p for g in self.param_groups for p in g["params"]], self.max_norm)
            return super().step(closure)
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        runs = {}
        for k, g in enumerate(self.param_groups):
            if g.get("amsgrad"):
                raise _lib.AyoloError("ayolov2_amd.optim.AdamW: amsgrad has no kernel")
            lr, ps = g["lr"], g["params"]
            if torch.is_tensor(lr) and not lr.is_cuda:
                lr = float(lr)
            # groups that differ in learning rate and decay alone share their launches
            key = (tuple(g["betas"]), g["eps"], bool(g["maximize"]), k if torch.is_tensor(lr) else -1)
            grads = [p.grad for p in ps]
            states = self._states(ps, grads)
            if key not in runs:
                runs[key] = ([], [], [], [], [], [], [])
            for l, more in zip(runs[key], (ps, grads, *states, [lr] * len(ps), [g["weight_decay"]] * len(ps))):
                l += more
        norm = grad_norm([g for run in runs.values() for g in run[1]], scale) if self.max_norm is not None else None
        if norm is not None and not norm.is_cuda:
            return loss                                    # no gradients at all
        for r, (key, (ps, grads, ms, vs, ts, lrs, wds)) in enumerate(runs.items()):
            # the seeds of several runs differ, so that their roundings do not repeat one another's
            _adamw(ps, grads, ms, vs, ts, lambda which, a=(ps, ms, vs): self._relay(*a, which), lrs[0] if key[3] >= 0 and lrs else lrs, key[0],
                   key[1], wds, key[2], self.seed + 0x51F15EED * r, norm, self.max_norm, scale, found)
        return loss

    def _check_states(self, state_dict) -> None:
        """Refuses a state dict whose states do not fit this optimiser's parameters."""
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            return                                         # the base class says what is wrong
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip((i for g in groups for i in g["params"]), params):
            raw = state_dict["state"].get(i)
            if not raw:
                continue
            what = f"ayolov2_amd.optim.AdamW: the state of parameter {i}"
            bits8 = "exp_avg_exps" in raw
            if bits8 and not p.is_cuda:
                raise _lib.AyoloError("ayolov2_amd.optim.AdamW: 8-bit states need parameters on the GPU")
            if not p.is_cuda:
                continue
            if self.state_bits == 8 and not bits8:
                raise _lib.AyoloError("ayolov2_amd.optim.AdamW: a state dict with 32-bit moments does not load into 8-bit states")
            for name in ("step", "exp_avg", "exp_avg_sq", *(("exp_avg_exps", "exp_avg_sq_exps") if bits8 else ())):
                if name not in raw:
                    raise _lib.AyoloError(f"{what} has no {name}")
            if torch.as_tensor(raw["step"]).numel() != 1:
                raise _lib.AyoloError(f"{what}: step is not one number")
            for name in ("exp_avg", "exp_avg_sq"):
                m = raw[name]
                if not torch.is_tensor(m) or m.shape != p.shape:
                    raise _lib.AyoloError(f"{what}: {name} is not a tensor of the parameter's shape {tuple(p.shape)}")
                if not bits8:
                    continue
                e = raw[name + "_exps"]
                if m.dtype != torch.uint8 or _layouts([m])[0] == 0:
                    raise _lib.AyoloError(f"{what}: {name} is not a dense block of 8-bit codes")
                if not torch.is_tensor(e) or e.dtype != torch.uint8 or e.shape != (-(-p.numel() // MOMENT_BLOCK),):
                    raise _lib.AyoloError(f"{what}: {name}_exps is not one byte per {MOMENT_BLOCK} codes")

    def load_state_dict(self, state_dict):
        # Hooks may hand on another state dict, and may change the loaded states: the check sees what all others before the load have
        # made of it, and the states are in place before the first hook behind it.
        seen = []

        def check(_, sd):
            self._check_states(sd)                         # before anything has changed
            seen.append(sd)

        hooks = (self.register_load_state_dict_pre_hook(check),
                 self.register_load_state_dict_post_hook(lambda _: self._take_states(seen[-1]), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()

    def _take_states(self, state_dict) -> None:
        """The states as they were saved (the base class has cast every one to its parameter's type)."""
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
            raw = state_dict["state"].get(i)
            if not raw or not p.is_cuda:
                continue
            st = self.state[p]
            st["step"] = torch.as_tensor(raw["step"], dtype=torch.float32).detach().reshape(()).to(p.device, copy=True)
            for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
                if "exp_avg_exps" in raw:
                    m = Moment8(raw[name].to(p.device, copy=True), raw[name + "_exps"].to(p.device, copy=True))
                    if self.state_bits == 8:
                        st[name], st[name + "_exps"] = _moment8_like(p, m, signed)
                    else:
                        st[name] = _moment_like(p, unpack_moments([m], signed)[0])
                        st.pop(name + "_exps", None)
                else:
                    st[name] = _moment_like(p, raw[name])
