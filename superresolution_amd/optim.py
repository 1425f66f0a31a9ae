"""Optimizer operators over a list of tensors (include/srgen.h, "optimizer operators over a list of tensors").

The reference's loops hold their parameters as separate tensors: ``optim.AdamW(generator.parameters(), lr)``
(``train.py:270,274-275``), ``grad_norm(generator)`` (``train.py:23-28,96``) and ``clip_grad_norm_(generator.parameters(), 10)``
(``train.py:175``).  Here those lines run as a few launches over the whole list:

    from superresolution_amd import optim
    opt_g = optim.AdamW(generator.parameters(), lr=cfg.lr_g, max_grad_norm=cfg.grad_clip_norm)   # clips inside step()
    opt_d = optim.AdamW(discriminator.parameters(), lr=cfg.lr_d, state_bits=8)                   # moments in 8 bits
    g = optim.grad_norm(generator)                                                               # 0-dim device tensor
    optim.clip_grad_norm_(generator.parameters(), 10.0)

``training.FlatAdamW`` (the fused training steps' optimizer) re-points the parameters at one flat buffer; nothing is re-pointed
here, any address will do.  ROCm tensors only: there is no CPU fallback.
"""
from __future__ import annotations

import contextlib
import ctypes
import os
from array import array
from itertools import accumulate
from operator import attrgetter
from typing import List, Optional, Tuple

import torch
from torch.optim import optimizer as _torch_optimizer

from . import _lib, versions


class _NotBuilt:
    """Stands for an extension that is missing (the package can be imported to build it): raises where it is used."""

    def __init__(self, why: Exception):
        self._why = why

    def __getattr__(self, name):
        raise _lib.SrgenError(f"{os.path.join(os.path.dirname(_lib.CSRC), '_tensorlist.so')} is missing or does not fit the installed "
                              f"torch ({self._why}): run `python -c 'import __graft_entry__ as g; g.build()'`. There is no fallback path.")


try:
    from . import _tensorlist
except ImportError as e:
    _tensorlist = _NotBuilt(e)

BLOCK = 32            # SRGEN_OPT_BLOCK: elements that share one scale (8-bit moments)
CHUNK = 4096          # SRGEN_OPT_CHUNK: elements of one step counter

_raw_stream = torch._C._cuda_getCurrentRawStream      # torch.cuda.current_stream(dev).cuda_stream without the object
_capturing = torch._C._cuda_isCurrentStreamCapturing  # torch.cuda.is_current_stream_capturing()
_current_device = torch._C._cuda_getDevice            # torch.cuda.current_device(), the runtime initialised
_HERE = contextlib.nullcontext()
_CODE = {torch.float32: _lib.SRGEN_F32, torch.bfloat16: _lib.SRGEN_BF16, torch.float16: _lib.SRGEN_F16}
_TYPES = frozenset((torch.float32, torch.bfloat16))                  # of parameters and their gradients
_dtype_of, _device_of = attrgetter("dtype"), attrgetter("device")
_data_ptr = torch.Tensor.data_ptr
_numel = torch.Tensor.numel


def _stream(dev: torch.device) -> int:
    return _raw_stream(dev.index)


def _on(dev: torch.device):
    """``dev`` as the current device, for a launch."""
    return _HERE if _current_device() == dev.index else torch.cuda.device(dev)


def _up(n: int, to: int) -> int:
    return -(-n // to) * to


def _addr(a: array) -> int:
    return a.buffer_info()[0]


def _dense(t: torch.Tensor) -> bool:
    """Every element at an address of its own and no gaps: what an elementwise kernel may walk in storage order."""
    if t.numel() == 0:
        return True
    want = 1
    for size, stride in sorted((z for z in zip(t.shape, t.stride()) if z[0] != 1), key=lambda z: z[1]):
        if stride != want:
            return False
        want *= size
    return True


def _own_memory(tensors, what: str) -> None:
    for t in tensors:
        if t.layout != torch.strided:
            raise RuntimeError(f"{what}: strided tensors, got {t.layout}")
        if t.numel() and not t.data_ptr():
            raise RuntimeError(f"{what}: a {type(t).__name__} has no memory of its own: pass the tensor that it wraps")


def _one_device(tensors, what: str) -> torch.device:
    devs = set(map(_device_of, tensors))
    if len(devs) != 1 or next(iter(devs)).type != "cuda":
        raise RuntimeError(f"{what}: tensors of one ROCm device, got {sorted(map(str, devs))}; there is no CPU fallback")
    return next(iter(devs))


def _no_overlap(ptr: array, numel: array, code: array, what: str) -> None:
    """Refuses a list of tensors that are written where two of them share memory."""
    if not _tensorlist.apart(len(ptr), ptr, numel, code):
        raise RuntimeError(f"{what}: two of the tensors share memory (the same one twice?)")


# ---- moments -----------------------------------------------------------------------------------------------------------
class Moments:
    """First and second moments of a list of tensors in one buffer each, the part of every tensor padded to whole blocks of 32
    elements, and the step counters.  32 bits: ``exp_avg``, ``exp_avg_sq`` (fp32).  8 bits: ``exp_avg`` and ``root`` -- the
    square root of the second moment -- in ``float8_e4m3fn``, with a ``float8_e8m0fnu`` power of two for each block in
    ``exp_avg_scale`` / ``root_scale``.  The square root has half the second moment's range in powers of two, which is what
    lets four bits of exponent and a scale hold it."""

    def __init__(self, numels: List[int], bits: int, device: torch.device):
        if bits not in (8, 32):
            raise ValueError(f"moments of {bits} bits: 8 or 32")
        self.numels, self.bits = list(numels), bits
        sizes = [_up(n, BLOCK) for n in numels]
        self.offsets = [0, *accumulate(sizes)][:-1]
        self.total = sum(sizes)
        counters = [-(-n // CHUNK) for n in numels]
        self.counter0 = [0, *accumulate(counters)]
        self.step = torch.zeros(self.counter0[-1], dtype=torch.int32, device=device)
        self.device = self.step.device                     # (with its index)
        if bits == 32:
            self.exp_avg = torch.zeros(self.total, dtype=torch.float32, device=device)
            self.exp_avg_sq = torch.zeros(self.total, dtype=torch.float32, device=device)
            ptrs = (self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), None, None)
        else:
            def byte(n, value):
                return torch.full((n,), value, dtype=torch.uint8, device=device)
            self.exp_avg = byte(self.total, 0).view(torch.float8_e4m3fn)
            self.root = byte(self.total, 0).view(torch.float8_e4m3fn)
            self.exp_avg_scale = byte(self.total // BLOCK, 1).view(torch.float8_e8m0fnu)      # what zeros are packed with
            self.root_scale = byte(self.total // BLOCK, 1).view(torch.float8_e8m0fnu)
            ptrs = tuple(t.data_ptr() for t in (self.exp_avg, self.root, self.exp_avg_scale, self.root_scale))
        self._numel, self._offset = array("Q", self.numels), array("Q", self.offsets)
        self._sizes = _addr(self._numel), _addr(self._offset)
        chunks = self.counter0[-1]
        table = torch.empty((chunks, 4), dtype=torch.int32)                    # which chunk is where: of the sizes alone
        _lib.check(_lib.lib().srgen_adamw_chunk_table(len(self.numels), _addr(self._numel), _addr(self._offset), table.data_ptr(), chunks))
        self._table = table.to(device)
        need = ctypes.c_size_t()
        _lib.check(_lib.lib().srgen_total_norm_scratch_bytes(len(self.numels), self._sizes[0], need))
        self.norm_bytes = need.value
        self._c = _lib.srgen_moments(bits, 0, *ptrs, self.step.data_ptr(), self._table.data_ptr(), self.total, chunks)

    @property
    def nbytes(self) -> int:
        """Device memory of the moments (without the step counters)."""
        return self.total * 8 if self.bits == 32 else 2 * self.total + 2 * (self.total // BLOCK)

    def steps(self) -> List[int]:
        """Steps each tensor has taken (reads them back from the device)."""
        if not self.numels:
            return []
        host = self.step.cpu()
        return [int(host[c]) if n else 0 for c, n in zip(self.counter0, self.numels)]

    def set_steps(self, steps: List[int]) -> None:
        counts = [b - a for a, b in zip(self.counter0, self.counter0[1:])]
        self.step.copy_(torch.repeat_interleave(torch.tensor(steps, dtype=torch.int32), torch.tensor(counts)))

    def read(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """Both moments as fp32 buffers in the padded layout (8 bits: new ones; 32 bits: the buffers themselves)."""
        if self.bits == 32:
            return self.exp_avg, self.exp_avg_sq
        return unpack_moments(self.exp_avg, self.exp_avg_scale, self.root, self.root_scale, self.total)

    def write(self, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor) -> None:
        """Takes fp32 buffers in the padded layout (the padding has to be zero)."""
        for t in (exp_avg, exp_avg_sq):
            if t.dtype != torch.float32 or t.shape != (self.total,) or t.device != self.device or not t.is_contiguous():
                raise RuntimeError(f"Moments.write: flat contiguous fp32 buffers of {self.total} elements on {self.device}, got "
                                   f"{tuple(t.shape)} {t.dtype} on {t.device}")
        if self.bits == 32:
            self.exp_avg.copy_(exp_avg)
            self.exp_avg_sq.copy_(exp_avg_sq)
            return
        _pack_into(exp_avg, exp_avg_sq, self.exp_avg, self.exp_avg_scale, self.root, self.root_scale)

    def update(self, p: array, g: array, p_dtype: array, g_dtype: array, args: "_lib.srgen_adamw_args", stream: int) -> None:
        """One AdamW step of the list (addresses and type codes in the list's order; address 0: no gradient)."""
        if not len(p) == len(g) == len(p_dtype) == len(g_dtype) == len(self.numels):
            raise ValueError(f"Moments.update: an address and a type code for each of the {len(self.numels)} tensors")
        if (p.typecode, g.typecode, p_dtype.typecode, g_dtype.typecode) != ("Q", "Q", "i", "i"):
            raise TypeError("Moments.update: addresses as array('Q'), type codes as array('i')")
        self._update((_addr(p), _addr(g)), (_addr(p_dtype), _addr(g_dtype)), args, stream)

    def _update(self, pg, codes, args, stream: int) -> None:
        rc = _lib.lib().srgen_adamw_many(len(self.numels), *pg, *self._sizes, *codes, self._c, args, stream)
        if rc:
            _lib.check(rc)


def _pack_into(exp_avg, exp_avg_sq, m8, me, r8, re) -> None:
    with _on(exp_avg.device):
        _lib.check(_lib.lib().srgen_moments_pack(exp_avg.data_ptr(), exp_avg_sq.data_ptr(), exp_avg.numel(), m8.data_ptr(), me.data_ptr(),
                                                 r8.data_ptr(), re.data_ptr(), _stream(exp_avg.device)))


def pack_moments(exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor):
    """``(m, m_scale, r, r_scale)``: the moments (flat fp32) as ``Moments`` holds them in 8 bits -- e4m3 values of the first
    moment and of the second one's square root, rounded to nearest, with a power of two for each 32 elements; ``m`` and ``r``
    are padded with zeros to whole blocks.  Values that 8 bits hold come back from ``unpack_moments`` as they were."""
    dev = _one_device((exp_avg, exp_avg_sq), "pack_moments")
    for t in (exp_avg, exp_avg_sq):
        if t.dtype != torch.float32 or t.dim() != 1 or not t.is_contiguous() or t.shape != exp_avg.shape:
            raise RuntimeError(f"pack_moments: two flat contiguous fp32 tensors of one length, got {tuple(t.shape)} {t.dtype}")
    n = _up(exp_avg.numel(), BLOCK)
    m8, r8 = (torch.empty(n, dtype=torch.float8_e4m3fn, device=dev) for _ in range(2))
    me, re = (torch.empty(n // BLOCK, dtype=torch.float8_e8m0fnu, device=dev) for _ in range(2))
    _pack_into(exp_avg, exp_avg_sq, m8, me, r8, re)
    return m8, me, r8, re


def unpack_moments(m8: torch.Tensor, m_scale: torch.Tensor, r8: torch.Tensor, r_scale: torch.Tensor, numel: int):
    """``(exp_avg, exp_avg_sq)``: the first ``numel`` elements of 8-bit moments in fp32, the second moment squared."""
    dev = _one_device((m8, m_scale, r8, r_scale), "unpack_moments")
    numel = int(numel)
    if not 0 <= numel <= m8.numel():
        raise RuntimeError(f"unpack_moments: {numel} of {m8.numel()} elements")
    for t, want, dt in ((m8, m8.numel(), torch.float8_e4m3fn), (r8, m8.numel(), torch.float8_e4m3fn),
                        (m_scale, m8.numel() // BLOCK, torch.float8_e8m0fnu), (r_scale, m8.numel() // BLOCK, torch.float8_e8m0fnu)):
        if t.dtype != dt or t.dim() != 1 or not t.is_contiguous() or t.numel() != want or m8.numel() % BLOCK:
            raise RuntimeError(f"unpack_moments: flat contiguous e4m3 values in whole blocks of {BLOCK} and an e8m0 scale for each, "
                               f"got {tuple(t.shape)} {t.dtype}")
        if t.data_ptr() % 4 and dt == torch.float8_e4m3fn:
            raise RuntimeError("unpack_moments: values must be 4-byte aligned")
    m, v = (torch.empty(numel, dtype=torch.float32, device=dev) for _ in range(2))
    with _on(dev):
        _lib.check(_lib.lib().srgen_moments_unpack(m8.data_ptr(), m_scale.data_ptr(), r8.data_ptr(), r_scale.data_ptr(), m.data_ptr(),
                                                   v.data_ptr(), numel, _stream(dev)))
    return m, v


# ---- total norm, clipping ----------------------------------------------------------------------------------------------
def _tensor_list(tensors) -> List[torch.Tensor]:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _codes(tensors, what: str) -> array:
    try:
        return array("i", map(_CODE.__getitem__, map(_dtype_of, tensors)))
    except KeyError as e:
        raise RuntimeError(f"{what}: fp32, bf16 or fp16 tensors, got {e.args[0]}") from None


def _arrays(n: int):
    return array("Q", bytes(8 * n)), array("Q", bytes(8 * n)), array("i", bytes(4 * n))


def _listed(tensors: List[torch.Tensor], what: str):
    """(device, tensors, addresses, sizes, type codes); a tensor with gaps is taken as a contiguous copy."""
    if not tensors[0].is_cuda:
        _one_device(tensors, what)                                             # (raises)
    dev = tensors[0].device
    ptr, numel, code = _arrays(len(tensors))
    if not _tensorlist.tensors(tensors, dev.index, ptr, numel, code):
        _one_device(tensors, what)
        _own_memory(tensors, what)
        code = _codes(tensors, what)
        tensors = [t if t.is_contiguous() or _dense(t) else t.detach().contiguous() for t in tensors]
        ptr, numel = array("Q", map(_data_ptr, tensors)), array("Q", map(_numel, tensors))
    return dev, tensors, ptr, numel, code


def _norm_coef(dev: torch.device, ptr: array, numel: array, code: array, max_norm: float, out: Optional[int] = None) -> torch.Tensor:
    """A device buffer that ends with {norm, clip coefficient}, or they go to the address ``out``; tensor address 0: left out."""
    L, need = _lib.lib(), ctypes.c_size_t()
    _lib.check(L.srgen_total_norm_scratch_bytes(len(ptr), _addr(numel), need))
    words = need.value // 4
    buf = torch.empty(words + 2, dtype=torch.float32, device=dev)              # partial sums, then {norm, coefficient}
    with _on(dev):
        _lib.check(L.srgen_total_norm(len(ptr), _addr(ptr), _addr(numel), _addr(code), max_norm, out or buf.data_ptr() + need.value, buf.data_ptr(),
                                      need.value, _stream(dev)))
    return buf


def total_norm(tensors) -> torch.Tensor:
    """The L2 norm of all ``tensors`` (fp32, bf16, fp16) taken together, as a 0-dim fp32 device tensor
    (``torch.nn.utils.get_total_norm``; not differentiable).  Sums are held in 64 bits and added in a fixed order: the result does
    not overflow before the norm itself does, and repeats bit for bit."""
    ts = _tensor_list(tensors)
    if not ts:
        return torch.tensor(0.0)
    dev, ts, ptr, numel, code = _listed(ts, "total_norm")
    return _norm_coef(dev, ptr, numel, code, 1.0)[-2]


def _grads(parameters) -> List[torch.Tensor]:
    if isinstance(parameters, torch.nn.Module):
        parameters = parameters.parameters()
    return [g for g in (p.grad for p in _tensor_list(parameters)) if g is not None]


def grad_norm(model) -> torch.Tensor:
    """``grad_norm(model)`` of the reference's loops (``train.py:23-28``): the L2 norm of all gradients of a module (or of an
    iterable of parameters), as a 0-dim device tensor instead of a Python float -- no synchronisation."""
    return total_norm(_grads(model))


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    foreach: Optional[bool] = None) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` (``train.py:175``): scales the gradients (of one device) in place so that their total L2
    norm is at most ``max_norm``; returns the norm before.  ``foreach`` is taken and has no meaning here.
    ``AdamW(max_grad_norm=...)`` clips without the extra pass."""
    if float(norm_type) != 2.0:
        raise NotImplementedError(f"clip_grad_norm_: the L2 norm only, got norm_type={norm_type}")
    grads = _grads(parameters)
    if not grads:
        return torch.tensor(0.0)
    dev, listed, ptr, numel, code = _listed(grads, "clip_grad_norm_")
    for g, t in zip(grads, listed):
        if g is not t:
            raise RuntimeError(f"clip_grad_norm_: a gradient of shape {tuple(g.shape)} and strides {g.stride()} has gaps or overlaps")
    _no_overlap(ptr, numel, code, "clip_grad_norm_")
    out = _norm_coef(dev, ptr, numel, code, float(max_norm))[-2:]
    if error_if_nonfinite and not bool(torch.isfinite(out[0])):
        raise RuntimeError("The total norm of order 2.0 for gradients from `parameters` is non-finite, so it cannot be clipped. To "
                           "disable this error and scale the gradients by the non-finite norm anyway, set `error_if_nonfinite=False`")
    with _on(dev):
        _lib.check(_lib.lib().srgen_scale_many(len(grads), _addr(ptr), _addr(numel), _addr(code), out.data_ptr() + 4, _stream(dev)))
    _tensorlist.bump(grads, None)
    return out[0]


# ---- AdamW -------------------------------------------------------------------------------------------------------------
_GLOBAL_HOOKS = (_torch_optimizer._global_optimizer_pre_hooks, _torch_optimizer._global_optimizer_post_hooks)


class _Lists:
    """A group's addresses and type codes, as the kernels' list wants them; filled anew at every step."""

    def __init__(self, params: List[torch.Tensor], seed: int):
        self.seed = seed
        self.p, self.g, self.p_code = _arrays(len(params))
        self.g_code = array("i", self.p_code)
        self.pg, self.codes = (_addr(self.p), _addr(self.g)), (_addr(self.p_code), _addr(self.g_code))
        self.checked = (array("Q"), array("i"))            # parameters' addresses and types that were last found apart
        self.shapes = [(p.shape, p.stride()) for p in params]          # as the moments have them
        self.order = [_order(p) for p in params]
        self.plain = all(p.is_contiguous() for p in params)


def _order(t: torch.Tensor) -> tuple:
    """The order of ``t``'s elements in memory: its strides, without those of axes of one element."""
    return () if t.numel() < 2 else tuple((n, a) for n, a in zip(t.shape, t.stride()) if n != 1)


def _in_order_of(p: torch.Tensor, g: torch.Tensor) -> torch.Tensor:
    """``g`` with its elements in the order of ``p``'s memory."""
    if g.shape != p.shape:
        raise RuntimeError(f"AdamW: a gradient of shape {tuple(g.shape)} for a parameter of shape {tuple(p.shape)}")
    if _order(g) == _order(p) and not g.is_neg():
        return g
    return torch.empty_strided(p.shape, p.stride(), dtype=g.dtype, device=g.device).copy_(g)


def group_seed(seed: int, group: int) -> int:
    """The seed of a group's random bits: positions count from 0 in every group's moments, and equal ones would round alike."""
    return (seed + group * 0x9E3779B9) & 0xFFFFFFFF


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` over separate tensors, a whole parameter group in one or a few launches.

    Parameters are fp32 or bf16 on one ROCm device, gradients either; arithmetic is fp32 (moments of 8 bits: 64 bits, then
    rounded).  Beyond torch's arguments:

    ``state_bits``      32: fp32 moments.  8: both moments in 8 bits (``Moments``), 2.06 bytes a parameter instead of 8, rounded
                        stochastically, so that a moving average goes on moving when its change is under half a step.
    ``max_grad_norm``   clips the gradients of all groups by their total norm inside ``step`` (the gradients themselves stay as
                        they are); the norm is left in ``last_grad_norm``.
    ``seed``            of the stochastic rounding, which depends on it, the step, the group and the element only (optimizers that
                        train side by side take seeds of their own, or elements at the same place round with the same bits).

    A bf16 parameter is rounded stochastically.  ``lr`` may be a 0-dim fp32 tensor on the parameters' device: a captured step
    then follows it, and ``load_state_dict`` writes into it (before a capture it makes a new one, as torch does).  Parameters keep
    the memory order that they were added with (``to(memory_format=...)`` comes before the optimizer).  ``step`` can be captured into a graph (the step counts are on the device); parameters, gradients and the
    optimizer have to stay.  While it does, ``Generator`` and ``Discriminator`` take its parameters for changed at every use (a replay
    raises no version counter, ``versions``).  ``torch.amp.GradScaler`` hands its scale and its flag to ``step``: a step with a non-finite
    gradient does not happen.  ``state_dict`` has the layout of ``torch.optim.AdamW`` with fp32 moments, whatever
    ``state_bits``: checkpoints move between the two, and between 8 and 32 bits (``state`` stays empty: ``moments`` has one
    ``Moments`` for each group).

    The random bits do not depend on the process: data-parallel ranks that take the same gradients stay the same bit for bit.
    A second moment beyond fp32's range (gradients of some 1e20) is infinite with 32 bits, which stops the element, and NaN with
    8.  Steps of one optimizer must not overlap, neither on two streams nor from two threads."""

    _step_supports_amp_scaling = True

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 max_grad_norm: Optional[float] = None, maximize: bool = False, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits={state_bits}: 8 or 32")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError(f"max_grad_norm={max_grad_norm}: positive, or None")
        self.state_bits, self.seed = state_bits, int(seed) & 0xFFFFFFFF
        self.max_grad_norm = None if max_grad_norm is None else float(max_grad_norm)
        self._norm_coef: Optional[torch.Tensor] = None     # ends with {norm, clip coefficient} of the last eager step
        # the same of every step from the first captured one on: a replay writes where the capture did, and the host does not see it
        self._norm_fixed: Optional[torch.Tensor] = None
        self._captured = False                             # a step has been captured
        self.moments: List[Moments] = []
        self._lists: List[_Lists] = []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        g = self.param_groups[-1]
        try:
            _check_hyper(g)
            dev = _one_device([p for h in self.param_groups for p in h["params"]], "AdamW")
            _own_memory(g["params"], "AdamW")
            for p in g["params"]:
                if p.dtype not in _TYPES:
                    raise RuntimeError(f"AdamW: fp32 or bf16 parameters, got {p.dtype}")
                if not _dense(p):
                    raise RuntimeError(f"AdamW: a parameter of shape {tuple(p.shape)} and strides {p.stride()} has gaps or overlaps")
            if len({id(p) for p in g["params"]}) != len(g["params"]):
                raise ValueError("AdamW: a parameter appears twice in a group")
            self._check_memory()
            # (allocated here and not at the first step: a first step inside a capture would put them into the graph's memory)
            if self._norm_fixed is None:
                self._norm_fixed = torch.full((2,), -1.0, dtype=torch.float32, device=dev)      # (-1: nothing yet)
            mo = Moments([p.numel() for p in g["params"]], self.state_bits, dev)
            ls = _Lists(g["params"], group_seed(self.seed, len(self._lists)))
        except BaseException:
            self.param_groups.pop()
            raise
        self.moments.append(mo)
        self._lists.append(ls)

    def _check_groups(self) -> None:
        if len(self.param_groups) != len(self.moments):
            raise RuntimeError(f"AdamW: {len(self.param_groups)} parameter groups, moments of {len(self.moments)}: groups come through "
                               "add_param_group, and stay")

    @property
    def last_grad_norm(self) -> Optional[torch.Tensor]:
        """The gradients' total norm at the last step that clipped, eager or replayed, before clipping (0-dim device tensor; NaN
        where a step has been captured and none has run)."""
        if not self._captured or self.max_grad_norm is None:
            return None if self._norm_coef is None else self._norm_coef[-2]
        # (a new tensor: the next step writes the buffer)
        norm = self._norm_fixed[0]
        return norm.masked_fill(norm < 0, float("nan")) if self._norm_coef is None else torch.where(norm < 0, self._norm_coef[-2], norm)

    # -- one step -----------------------------------------------------------------------------------------------------
    def step(self, closure=None):
        # torch wraps the step() of every optimizer in a profiler range and its hooks, which takes longer than a small step does:
        # here only where a profiler runs or somebody has registered a hook
        try:
            if (torch._C._autograd._profiler_enabled() or self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks
                    or any(_GLOBAL_HOOKS)):
                return self._step_with_hooks(closure)
            return self._step(closure)
        except BaseException:
            # GradScaler takes these back only after a step that returns: a later step would divide by this one's scale
            self.__dict__.pop("grad_scale", None)
            self.__dict__.pop("found_inf", None)
            raise

    step.hooked = True                                     # (how torch's wrapper marks the ones it has wrapped)

    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if len(self.param_groups) != len(self.moments):
            self._check_groups()
        counts, kept = [], []
        for k, (group, mo, ls) in enumerate(zip(self.param_groups, self.moments, self._lists)):
            n = _tensorlist.params(group["params"], mo.device.index, mo._numel, ls.p, ls.p_code, ls.g, ls.g_code)
            if n < 0 or not ls.plain:
                n = self._look_closer(k, kept)
            if ls.p != ls.checked[0] or ls.p_code != ls.checked[1]:
                self._check_memory()
            counts.append(n)
        if not any(counts):
            return loss
        dev = self.moments[0].device
        div, found = self.__dict__.get("grad_scale"), self.__dict__.get("found_inf")
        for t in (div, found):
            if t is not None and (t.device != dev or t.dtype != torch.float32 or t.numel() != 1):
                raise RuntimeError(f"AdamW: grad_scale and found_inf are fp32 scalars on {dev}")
        if self.max_grad_norm is not None and div is not None:
            raise RuntimeError("AdamW(max_grad_norm=...) clips the gradients as they are: call scaler.unscale_(optimizer) before "
                               "scaler.step(optimizer)")
        calls = []                                         # (all of them before the first: no group steps if another is refused)
        for n, group, mo, ls in zip(counts, self.param_groups, self.moments, self._lists):
            if not n:
                continue
            lr, (b1, b2) = group["lr"], group["betas"]
            lr_dev = None
            if isinstance(lr, torch.Tensor):
                if lr.is_cuda:
                    if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != dev:
                        raise RuntimeError(f"AdamW: a learning rate on the device is an fp32 scalar on {dev}")
                    lr_dev, lr = lr.data_ptr(), 0.0
                else:
                    lr = float(lr)
            if len(counts) > 1:                            # (one group: the library refuses it)
                _check_hyper({**group, "lr": lr})
            calls.append((group, mo, ls, _lib.srgen_adamw_args(
                lr, b1, b2, group["eps"], group["weight_decay"], lr_dev, None, None if div is None else div.data_ptr(),
                None if found is None else found.data_ptr(), None, None, mo.norm_bytes, self.max_grad_norm or 0.0, ls.seed,
                1 if group["maximize"] else 0)))
        with _on(dev):
            stream, capturing = _stream(dev), _capturing()
            norm_coef = fixed = None
            if self.max_grad_norm is not None:
                if capturing or self._captured:
                    fixed = self._norm_fixed.data_ptr()
                if len(counts) == 1:                       # norm and step in one call
                    mo, args = self.moments[0], calls[0][3]
                    norm_coef = torch.empty(mo.norm_bytes // 4 + 2, dtype=torch.float32, device=dev)
                    args.norm_scratch = norm_coef.data_ptr()
                    args.norm_coef2 = fixed or args.norm_scratch + mo.norm_bytes
                else:
                    g, numel, code = array("Q"), array("Q"), array("i")
                    for mo, ls in zip(self.moments, self._lists):
                        g, numel, code = g + ls.g, numel + mo._numel, code + ls.g_code
                    norm_coef = _norm_coef(dev, g, numel, code, self.max_grad_norm, fixed)
                    for *_, args in calls:
                        args.grad_mul = (fixed or norm_coef.data_ptr() + 4 * (norm_coef.numel() - 2)) + 4
            for group, mo, ls, args in calls:
                mo._update(ls.pg, ls.codes, args, stream)
                # the kernel wrote behind torch's back: the version counters are what the Generator / Discriminator mirrors
                # watch to upload their weights again
                _tensorlist.bump(group["params"], ls.g)
            if capturing:                                  # (its replays will write them, and raise no counter)
                self._captured = True
                for group, _, ls, _ in calls:
                    versions.note_captured((p for p, g in zip(group["params"], ls.g) if g), self)
        if norm_coef is not None and not fixed:            # (a refused step leaves the last one's)
            self._norm_coef = norm_coef
        return loss

    _step_with_hooks = torch.optim.Optimizer.profile_hook_step(_step)

    @torch.no_grad()
    def _look_closer(self, k: int, kept: list) -> int:
        """Group ``k`` has a tensor that is not plain (contiguous fp32 or bf16, on the device, of the size it was added with):
        refused, or its gradient brought into the parameter's order; such copies are put into ``kept``."""
        params, mo, ls = self.param_groups[k]["params"], self.moments[k], self._lists[k]
        if list(map(_numel, params)) != mo.numels:
            raise RuntimeError("AdamW: a parameter has another number of elements than when it was added")
        grads = [p.grad for p in params]
        some = [g for g in grads if g is not None]
        for what, ts in (("parameters", params), ("gradients", some)):
            if not _TYPES.issuperset(map(_dtype_of, ts)):
                raise RuntimeError(f"AdamW: fp32 or bf16 {what}, got {sorted({str(t.dtype) for t in ts})}")
            if any(t.device != mo.device for t in ts):
                raise RuntimeError(f"AdamW: {what} that are not on {mo.device}, where the moments are")
            _own_memory(ts, f"AdamW: {what}")
        for p, order in zip(params, ls.order):
            if p.is_neg():
                raise RuntimeError("AdamW: a parameter that is a lazily negated view")
            # (the number of elements is known; a shape of the same order, flattened or with other axes, is the same memory)
            if _order(p) != order and not (p.is_contiguous() and ls.plain):
                raise RuntimeError(f"AdamW: a parameter of shape {tuple(p.shape)} and strides {p.stride()}: its memory had another "
                                   "order when it was added, which its moments still have")
        grads = [g if g is None else _in_order_of(p, g) for p, g in zip(params, grads)]
        kept += grads
        ls.p[:] = array("Q", map(_data_ptr, params))
        ls.p_code[:] = _codes(params, "AdamW")
        ls.g[:] = array("Q", [0 if g is None else g.data_ptr() for g in grads])
        ls.g_code[:] = array("i", [0 if g is None else _CODE[g.dtype] for g in grads])
        return len(some)

    def _check_memory(self) -> None:
        """No two parameters share memory: looked at when their addresses are not those that were looked at last."""
        seen = [(array("Q", map(_data_ptr, h["params"])), array("Q", map(_numel, h["params"])), _codes(h["params"], "AdamW"))
                for h in self.param_groups]
        every = [array(t) for t in "QQi"]
        for ptr, numel, code in seen:
            for a, b in zip(every, (ptr, numel, code)):
                a.extend(b)
        _no_overlap(*every, "AdamW")
        for ls, (ptr, _, code) in zip(self._lists, seen):
            ls.checked = ptr, code

    # -- checkpoints --------------------------------------------------------------------------------------------------
    def _places(self, k: int) -> list:
        """(shape, strides, offset) of each tensor of group ``k`` in the moments' buffers, by the order that the parameter was added
        with; its present shape where that is the same memory."""
        params, mo, ls = self.param_groups[k]["params"], self.moments[k], self._lists[k]
        if list(map(_numel, params)) != mo.numels:
            raise RuntimeError("AdamW: a parameter has another number of elements than when it was added")
        places = []
        for p, (shape, stride), offset in zip(params, ls.shapes, mo.offsets):
            if p.shape != shape:
                if not p.is_contiguous() or not ls.plain:
                    raise RuntimeError(f"AdamW: a parameter of shape {tuple(p.shape)} and strides {p.stride()}: it was added with shape "
                                       f"{tuple(shape)} and strides {stride}, which its moments still have")
                shape, stride = p.shape, p.stride()
            places.append((shape, stride, offset))
        return places

    def state_dict(self) -> dict:
        """``torch.optim.AdamW.state_dict()``'s layout (``train.py:219-225`` saves it): fp32 moments and a step for each
        parameter that has taken one.  Reads the step counts back: one synchronisation."""
        for hook in self._optimizer_state_dict_pre_hooks.values():
            hook(self)
        self._check_groups()
        state, groups, first = {}, [], 0
        for k, (group, mo) in enumerate(zip(self.param_groups, self.moments)):
            m, v = mo.read()
            for i, (p, t, place) in enumerate(zip(group["params"], mo.steps(), self._places(k))):
                if t:
                    state[first + i] = {"step": torch.tensor(float(t)), **{
                        key: torch.empty_strided(p.shape, p.stride(), dtype=torch.float32, device=mo.device).copy_(
                            torch.as_strided(x, *place)) for key, x in (("exp_avg", m), ("exp_avg_sq", v))}}
            groups.append({**{k: x.detach().clone() if isinstance(x, torch.Tensor) else x for k, x in group.items() if k != "params"},
                           "params": list(range(first, first + len(group["params"])))})
            first += len(group["params"])
        sd = {"state": state, "param_groups": groups}
        for hook in self._optimizer_state_dict_post_hooks.values():
            given = hook(self, sd)
            sd = sd if given is None else given
        return sd

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict) -> None:
        """Takes what ``state_dict`` (of this class, whatever its ``state_bits``, of ``torch.optim.AdamW`` or of
        ``training.FlatAdamW``) returns."""
        state_dict = state_dict.copy()
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            given = hook(self, state_dict)
            state_dict = state_dict if given is None else given
        self._check_groups()
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("loaded state dict contains a parameter group that doesn't match the size of optimizer's group")
        state = state_dict["state"]
        if any(g.get("amsgrad") for g in groups):
            raise ValueError("AdamW: no amsgrad variant")
        if not all(g.get("decoupled_weight_decay", True) for g in groups):
            raise ValueError("AdamW: no variant that adds the weight decay to the gradient")
        plan = []                                          # (every group is looked at before the first is written)
        for k, (group, saved) in enumerate(zip(self.param_groups, groups)):
            for p, key in zip(group["params"], saved["params"]):
                for name in ("exp_avg", "exp_avg_sq"):
                    if key in state and state[key][name].numel() != p.numel():
                        raise ValueError(f"optimizer state of parameter {key} has {state[key][name].numel()} entries, the parameter {p.numel()}")
            _check_hyper({**group, **{k: x for k, x in saved.items() if k != "params"}})
            plan.append((self._places(k), [int(float(state[key]["step"])) if key in state else 0 for key in saved["params"]]))
        if self._captured:
            shared = {}                                    # scalars that are written in place
            for group, saved in zip(self.param_groups, groups):
                lr, value = group["lr"], saved.get("lr", group["lr"])
                if isinstance(lr, torch.Tensor) and lr.is_cuda:
                    value = torch.as_tensor(value).to(lr).reshape(())
                    if not torch.equal(shared.setdefault(lr.data_ptr(), value), value):
                        raise ValueError("AdamW: groups share a learning rate that a captured step reads, and the checkpoint has two for it")
        for (group, mo, saved), (places, steps) in zip(zip(self.param_groups, self.moments, groups), plan):
            m = torch.zeros(mo.total, dtype=torch.float32, device=mo.device)
            v = torch.zeros_like(m)
            into, values = [], []
            for place, key in zip(places, saved["params"]):
                st = state.get(key)
                if st is not None:
                    for x, name in ((m, "exp_avg"), (v, "exp_avg_sq")):
                        into.append(torch.as_strided(x, *place))
                        values.append(st[name].detach().reshape(place[0]))
            if into:
                torch._foreach_copy_(into, values)
            if steps:
                mo.set_steps(steps)
            mo.write(m, v)
            lr = self._loaded_lr(group["lr"], saved.get("lr", group["lr"]))
            group.update({k: x.clone() if isinstance(x, torch.Tensor) else x for k, x in saved.items() if k not in ("params", "lr")}, lr=lr)
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    def _loaded_lr(self, lr, saved):
        """What a group's learning rate becomes: a scalar on the device stays one, and the very one that a captured step reads."""
        if isinstance(lr, torch.Tensor) and lr.is_cuda:
            saved = torch.as_tensor(saved).reshape(lr.shape)
            return lr.copy_(saved) if self._captured else torch.empty_like(lr).copy_(saved)
        return saved.clone() if isinstance(saved, torch.Tensor) else saved

    def __getstate__(self):
        raise RuntimeError("AdamW holds device buffers: save state_dict() instead of the optimizer")


def _check_hyper(g: dict) -> None:
    b1, b2 = g["betas"]
    if isinstance(g["lr"], torch.Tensor):
        if g["lr"].numel() != 1:
            raise ValueError("Tensor lr must be 1-element")
    elif not g["lr"] >= 0.0:
        raise ValueError(f"Invalid learning rate: {g['lr']}")
    if not g["eps"] >= 0.0:
        raise ValueError(f"Invalid epsilon value: {g['eps']}")
    if not g["weight_decay"] >= 0.0:
        raise ValueError(f"Invalid weight_decay value: {g['weight_decay']}")
    for i, b in enumerate((b1, b2)):
        if not 0.0 <= b < 1.0:
            raise ValueError(f"Invalid beta parameter at index {i}: {b}")
