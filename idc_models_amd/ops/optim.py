"""Fused optimizer entry points (native HIP kernels over flat fp32 arenas or many tensors).

``rmsprop_`` updates one flat arena.  The AdamW step and the global norm of the gradients take a
``TensorTable``, which describes any number of tensors once, so that a call is one to three launches:

    table = TensorTable(grads, params, decay=[p.dim() > 1 for p in params])
    state = AdamWState(table, bits=8)
    adamw_(table, state, lr=1e-3, weight_decay=0.01, clip_norm=1.0)

Calls go to the current stream of the tensors' device, allocate nothing but ``global_norm``'s
result and workspace, and can be captured in a HIP graph (the step counter lives on the device).
Two calls that change one state, or one call and a change of its gradients, have to be ordered by the caller.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from . import _native as nat
from . import moments8

_MIN, _MAX = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max
_CHUNK = np.dtype([("w", "u8"), ("g", "u8"), ("base", "i8"), ("n", "i4"), ("flags", "i4")])


def rmsprop_(w: torch.Tensor, g: torch.Tensor, ms: torch.Tensor, lr: float, rho: float, eps: float,
             grad_scale: float = 1.0) -> None:
    """Keras RMSprop in place: ms = rho*ms + (1-rho)*(s*g)^2; w -= lr*s*g/(sqrt(ms)+eps)."""
    assert w.is_cuda and w.dtype == torch.float32 and w.numel() % 4 == 0
    nat.require().rmsprop(w.data_ptr(), g.data_ptr(), ms.data_ptr(), w.numel(), float(lr), float(rho),
                          float(eps), float(grad_scale), nat.stream_handle())


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one stretch of memory, each place once, in any order of the axes."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.numel() == 0 or all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def _span(t: torch.Tensor) -> Tuple[int, int]:
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


class _Held:
    """The memory at addresses that are read once.  A tensor object does not hold it: ``p.data = x`` (and what
    does that: ``Module.to``, the arena that ``Model.compile`` makes) gives the same object other storage and
    frees the first one.  So each tensor's storage is kept, and ``moved`` says whether one of the objects
    lies elsewhere by now."""

    def __init__(self, tensors: Sequence[torch.Tensor]):
        self.tensors = list(tensors)
        self.memory = [t.untyped_storage() for t in self.tensors]  # (0.14 us each; an alias, detach(): 0.6)
        self.at, self.every = [t.data_ptr() for t in self.tensors], list(range(len(self.tensors)))

    def moved(self) -> bool:
        # one call into torch: 0.1 us for a tensor, 16 for 600 (data_ptr() in Python: 0.13 and 24)
        return not torch._C._tensors_data_ptrs_at_indices_equal(self.tensors, self.at, self.every)

    def changed(self) -> None:
        """Tells autograd that a kernel has written to the tensors: a backward pass through a graph that saved
        them raises, as after any operation in place."""
        torch.autograd.graph.increment_version(self.tensors)


def chunk_size(sizes: Sequence[int]) -> int:
    """Elements of a full piece of a table (csrc/kernels/adamw.h)."""
    return nat.OPT_CHUNK_BIG if sum(sizes) >= nat.OPT_MAX_GRID * nat.OPT_CHUNK_BIG else nat.OPT_CHUNK


def chunk_table(sizes: Sequence[int], w_ptrs: Sequence[int], g_ptrs: Sequence[int], grad_bytes: int,
                decay: Sequence[bool], chunk: int) -> Tuple[np.ndarray, np.ndarray, int]:
    """``(pieces, offsets, numel)``: the OptChunk records (of at most ``chunk`` elements) of tensors with
    these sizes and addresses, every tensor's place in the flat state (multiples of 64), and the state's length."""
    n = np.asarray(sizes, dtype=np.int64)
    room = (n + nat.OPT_BLOCK - 1) // nat.OPT_BLOCK * nat.OPT_BLOCK
    offsets = np.concatenate([[0], np.cumsum(room)])
    w, g = np.asarray(w_ptrs, dtype=np.uint64), np.asarray(g_ptrs, dtype=np.uint64)
    vec = (w % 16 == 0) & (g % 16 == 0)
    flags = np.asarray(decay, dtype=bool) * nat.OPT_DECAY + vec * nat.OPT_VEC
    count = (n + chunk - 1) // chunk
    of = np.repeat(np.arange(len(n)), count)  # the tensor of every piece
    start = (np.arange(len(of)) - np.repeat(np.cumsum(count) - count, count)) * chunk
    out = np.zeros(len(of), dtype=_CHUNK)
    out["w"] = np.where(w[of] != 0, w[of] + (start * 4).astype(np.uint64), 0)
    out["g"] = g[of] + (start * grad_bytes).astype(np.uint64)
    out["base"] = offsets[:-1][of] + start
    out["n"] = np.minimum(n[of] - start, chunk)
    out["flags"] = flags[of]
    return out, offsets[:-1], int(offsets[-1])


class TensorTable:
    """The tensors of a multi-tensor launch: gradients (fp32, or all bf16) and, for an optimizer step,
    the fp32 weights they belong to.

    The addresses are read here once: gradients have to be accumulated in place afterwards, as an
    arena's are, and weights have to keep their storage.  Where it is replaced (``p.data = x``,
    ``Module.to``, ``Model.compile``, which moves a model's weights into an arena), a new table is needed: ``adamw_``
    refuses weights that are Parameters or require a gradient, ``check`` any tensor.  The table keeps the first
    storage alive, but resizing a listed tensor in place frees its memory all the same: not before the table's last
    call.  A weight and its gradient have the same shape and the same order of axes in memory, without
    gaps.  Empty tensors are fine.  ``decay``: which weights decay (default: all)."""

    def __init__(self, grads: Sequence[torch.Tensor], params: Optional[Sequence[torch.Tensor]] = None,
                 decay: Optional[Sequence[bool]] = None):
        grads = list(grads)
        params = None if params is None else list(params)
        if not grads:
            raise ValueError("TensorTable needs at least one tensor")
        every = grads + (params or [])
        if not all(isinstance(t, torch.Tensor) and t.layout == torch.strided for t in every):
            raise ValueError("TensorTable takes dense tensors")
        self.device, self.grad_dtype = grads[0].device, grads[0].dtype
        if self.grad_dtype not in (torch.float32, torch.bfloat16) or any(g.dtype != self.grad_dtype for g in grads):
            raise ValueError("gradients have to be all float32 or all bfloat16")
        if any(t.device != self.device for t in every):
            raise ValueError("all tensors have to be on one device")
        if not all(_dense(t) for t in every):
            raise ValueError("tensors with gaps, or with elements that share memory, are not supported")
        if params is None:
            if decay is not None:
                raise ValueError("decay needs params")
            decay = [False] * len(grads)
        else:
            if len(params) != len(grads):
                raise ValueError(f"{len(params)} params for {len(grads)} grads")
            if any(p.dtype != torch.float32 for p in params):
                raise ValueError("params have to be float32")
            for i, (p, g) in enumerate(zip(params, grads)):
                if p.shape != g.shape or not _same_order(p, g):
                    raise ValueError(f"param and grad {i} differ in shape or in the order of their axes")
            decay = [True] * len(params) if decay is None else [bool(d) for d in decay]
            if len(decay) != len(params):
                raise ValueError(f"{len(decay)} decay flags for {len(params)} params")
            spans = sorted(_span(p) for p in params if p.numel())
            if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
                raise ValueError("params overlap in memory")
            both = sorted([(*s, 0) for s in spans] + [(*_span(g), 1) for g in grads if g.numel()])
            reach = [0, 0]  # the furthest end so far of the params and of the grads
            for lo, hi, kind in both:
                if lo < reach[1 - kind]:
                    raise ValueError("params and grads overlap in memory")
                reach[kind] = max(reach[kind], hi)
        if self.device.type != "cuda":
            raise ValueError("TensorTable needs tensors on a GPU")
        self.grads, self.params = grads, params
        self._all = _Held(every)
        # (isinstance asks Parameter's metaclass: 0.4 us)
        leaves = [p for p in params or [] if p.requires_grad or issubclass(type(p), torch.nn.Parameter)]
        self._leaves = _Held(leaves) if leaves else None
        sizes = [g.numel() for g in grads]
        self.chunk = chunk_size(sizes)
        pieces, offsets, self.numel = chunk_table(
            sizes, [p.data_ptr() for p in params] if params is not None else [0] * len(grads),
            [g.data_ptr() for g in grads], self.grad_dtype.itemsize, decay, self.chunk)
        if len(pieces) >= 1 << 31:
            raise ValueError("too many elements for one table")
        self.sizes, self.offsets = sizes, offsets.tolist()
        self.nchunks = len(pieces)
        host = torch.from_numpy(pieces.view(np.uint8)) if self.nchunks else torch.zeros(1, dtype=torch.uint8)
        self.chunks = host.to(self.device)
        self._bf16 = int(self.grad_dtype == torch.bfloat16)

    def check(self) -> None:
        """Raises ValueError if any of the tensors has other storage than when the table was made."""
        if self._all.moved():
            raise ValueError("a tensor has other storage than when the table was made")

    def split(self, flat: torch.Tensor):
        """Views of a flat state tensor in the shapes of the table's contiguous tensors (others: flat
        views in their order in memory)."""
        return [flat[o:o + n].view(g.shape) if g.is_contiguous() else flat[o:o + n]
                for o, n, g in zip(self.offsets, self.sizes, self.grads)]


class AdamWState:
    """Moments and step counter of an AdamW step over a table's tensors, or over those of another table of
    tensors of the same sizes in the same order.

    ``bits=32``: ``m`` and ``v`` are fp32, ``table.numel`` long.  ``bits=8``: codes of the first moment
    and of the root of the second (uint8), and ``scales``, two bytes for 64 of them: 2.03 bytes a
    weight instead of 8.  ``step``: int32 copies of the number of steps done, all equal
    (``set_step``).  ``norm``: the global norm that the last clipped step saw."""

    def __init__(self, table: TensorTable, bits: int = 32):
        if bits not in (8, 32):
            raise ValueError(f"AdamW states have 8 or 32 bits, not {bits}")
        if table.params is None:
            raise ValueError("the table has no params")
        self.bits, self.numel, self.device, self.sizes = bits, table.numel, table.device, table.sizes
        dtype = torch.uint8 if bits == 8 else torch.float32
        room = max(self.numel, nat.OPT_BLOCK)  # a table of empty tensors still has a state
        self.m = torch.zeros(room, dtype=dtype, device=self.device)[:self.numel]
        self.v = torch.zeros(room, dtype=dtype, device=self.device)[:self.numel]
        self.scales = torch.zeros(room // nat.OPT_BLOCK, 2, dtype=torch.uint8,
                                  device=self.device)[:self.numel // nat.OPT_BLOCK] if bits == 8 else None
        self.step = torch.zeros(nat.OPT_MAX_GRID, dtype=torch.int32, device=self.device)
        self._work = torch.zeros(4, dtype=torch.float32, device=self.device)
        self.norm = self._work[0]
        self.partials = torch.zeros(nat.OPT_MAX_GRID, dtype=torch.float64, device=self.device)
        a = self._args = nat.AdamwArgs()
        a.m, a.v, a.scales = self.m.data_ptr(), self.v.data_ptr(), nat.ptr(self.scales)
        a.step, a.norm = self.step.data_ptr(), self._work.data_ptr()

    def tensors(self) -> dict:
        """What a checkpoint keeps."""
        out = {"m": self.m, "v": self.v, "step": self.step}
        if self.scales is not None:
            out["scales"] = self.scales
        return out

    def set_step(self, n: int) -> None:
        self.step.fill_(int(n))

    def reset(self) -> None:
        for t in self.tensors().values():
            t.zero_()

    def decode(self, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """The values an 8-bit state stands for: the first moments and the ROOTS of the second ones,
        flat (``table.split`` gives them shapes), in float32 or bfloat16 (both exact)."""
        if self.bits != 8:
            raise ValueError("decode is for 8-bit states")
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("decode gives float32 or bfloat16")
        m = torch.empty(self.numel, dtype=dtype, device=self.device)
        r = torch.empty_like(m)
        with _on(self.device):
            nat.require().adamw_decode(self.m.data_ptr(), self.v.data_ptr(), self.scales.data_ptr(), self.numel,
                                       m.data_ptr(), r.data_ptr(), int(dtype == torch.bfloat16),
                                       _stream(self.device))
        return m, r

    def moments(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """First and second moments, flat, fp32 (of a 32-bit state: its own tensors)."""
        if self.bits == 32:
            return self.m, self.v
        m, r = self.decode()
        return m, r * r

    def load_moments(self, m: torch.Tensor, v: torch.Tensor) -> None:
        """Takes flat fp32 moments (an 8-bit state rounds them to its nearest codes)."""
        if m.shape != self.m.shape or v.shape != self.v.shape:
            raise ValueError(f"moments of {tuple(m.shape)} and {tuple(v.shape)} for a state of {self.numel}")
        m, v = (t.to(self.device, torch.float32) for t in (m, v))
        if self.bits == 32:
            self.m.copy_(m)
            self.v.copy_(v)
        elif self.numel:
            self.m[:], self.scales[:, 0] = moments8.encode(m, moments8.M_BITS)
            self.v[:], self.scales[:, 1] = moments8.encode(v.sqrt(), moments8.ROOT_BITS)


class _Here:
    def __enter__(self):
        return self

    def __exit__(self, *a):
        return False


_HERE = _Here()


def _on(device: torch.device):
    """Launches go to the device that is current: the tensors' one has to be."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    # current_stream(device).cuda_stream builds a Stream object for its handle: 1.7 of a 6.7 us call
    return torch._C._cuda_getCurrentRawStream(device.index)


def check_adamw(lr: float, beta_1: float, beta_2: float, epsilon: float, weight_decay: float, clip_norm: float) -> None:
    """Raises ValueError for hyperparameters an AdamW step cannot run with."""
    if not (0.0 <= beta_1 < 1.0 and 0.0 <= beta_2 < 1.0):
        raise ValueError(f"betas have to be in [0, 1): {beta_1}, {beta_2}")
    if not (lr >= 0.0 and weight_decay >= 0.0 and max(lr, weight_decay, lr * weight_decay, epsilon) <= _MAX):
        raise ValueError(f"lr and weight_decay have to be finite and not negative: {lr}, {weight_decay}")
    if not (clip_norm == 0.0 or _MIN <= clip_norm <= _MAX):
        raise ValueError(f"clip_norm has to be 0 (no clipping) or a positive fp32 number: {clip_norm}")
    if not epsilon >= _MIN:
        # without it, every weight whose gradients have all been zero would become 0 / 0
        raise ValueError(f"epsilon has to be a positive fp32 number: {epsilon}")


def set_adamw_args(a: "nat.AdamwArgs", table: TensorTable, state: AdamWState, lr: float, beta_1: float, beta_2: float,
                   epsilon: float, weight_decay: float, grad_scale: float, clip_norm: float, skip: int = 0,
                   hostflag: int = 0) -> "nat.AdamwArgs":
    a.chunks, a.nchunks, a.chunk = table.chunks.data_ptr(), table.nchunks, table.chunk
    a.b1, a.b2, a.omb1, a.omb2 = beta_1, beta_2, 1.0 - beta_1, 1.0 - beta_2
    a.log_b1 = math.log(beta_1) if beta_1 else -math.inf
    a.log_b2 = math.log(beta_2) if beta_2 else -math.inf
    a.lr, a.eps, a.lr_wd = lr, epsilon, lr * weight_decay
    a.grad_scale, a.clip = grad_scale, clip_norm
    if clip_norm and table.nchunks > nat.OPT_OWN_SUM:  # grad_norm's partial sums; else the step sums by itself
        a.partials, a.npartials = state.partials.data_ptr(), min(table.nchunks, nat.OPT_MAX_GRID)
    else:
        a.partials, a.npartials = 0, 0
    a.skip, a.hostflag = skip, hostflag
    return a


def adamw_(table: TensorTable, state: AdamWState, lr: float, beta_1: float = 0.9, beta_2: float = 0.999,
           epsilon: float = 1e-7, weight_decay: float = 0.004, grad_scale: float = 1.0, clip_norm: float = 0.0,
           skip: Optional[torch.Tensor] = None) -> None:
    """One Keras AdamW step over the table's tensors, in place, in one launch (two from 33.5 million weights on):

        t += 1;  g = grad_scale * grad;  m = beta_1*m + (1-beta_1)*g;  v = beta_2*v + (1-beta_2)*g^2
        w -= lr*weight_decay*w + lr*sqrt(1-beta_2^t)/(1-beta_1^t) * m/(sqrt(v)+epsilon)

    ``clip_norm`` > 0 scales g down to that global norm (one launch more for all but small tables, nothing
    is read back; a norm that is not finite makes every gradient NaN).  ``skip``: an int32 tensor on the
    device; if its first word is not zero the call changes nothing.  The numbers are arguments of the
    launch: a captured call keeps those it was captured with, and counts its steps on the device.

    Autograd sees the change of weights that are Parameters or require a gradient (a replayed graph's changes
    it does not see): a second backward pass through a graph that saved them raises."""
    check_adamw(lr, beta_1, beta_2, epsilon, weight_decay, clip_norm)
    if not abs(grad_scale) <= _MAX:
        raise ValueError(f"grad_scale has to be finite: {grad_scale}")
    if table.params is None:
        raise ValueError("the table has no params")
    # every tensor's moments lie at its place (the first comparison is what a program meets that keeps its table)
    if (state.sizes is not table.sizes and state.sizes != table.sizes) or state.device != table.device:
        raise ValueError("the state was made for another table")
    leaves = table._leaves
    if leaves is not None and leaves.moved():
        raise ValueError("a weight has other storage than when the table was made")
    if skip is not None and (skip.dtype != torch.int32 or skip.device != table.device or not skip.numel()):
        raise ValueError("skip has to be an int32 tensor on the tensors' device")
    a = set_adamw_args(state._args, table, state, lr, beta_1, beta_2, epsilon, weight_decay, grad_scale, clip_norm,
                       nat.ptr(skip))
    ext = nat.require()
    with _on(table.device):
        stream = _stream(table.device)
        if a.partials:
            ext.grad_norm(a.chunks, table.nchunks, table._bf16, a.partials, 0, stream)
        ext.adamw(ctypes.addressof(a), state.bits, table._bf16, stream)
    if leaves is not None:
        leaves.changed()


def global_norm(table: TensorTable) -> torch.Tensor:
    """sqrt of the sum of the squares of all the table's gradients: an fp32 tensor without axes.
    Sums in a fixed order (the same bits every time), in fp64; of bf16 gradients up to 16 squares, exact
    in fp32, are summed there first, where none of them leaves its range."""
    dev = table.device
    many = table.nchunks > nat.OPT_NORM_ONE
    partials = torch.empty(nat.OPT_MAX_GRID, dtype=torch.float64, device=dev) if many else None
    out = torch.empty((), dtype=torch.float32, device=dev)
    ext = nat.require()
    with _on(dev):
        ext.grad_norm(table.chunks.data_ptr(), table.nchunks, table._bf16, nat.ptr(partials), out.data_ptr(),
                      _stream(dev))
    return out
