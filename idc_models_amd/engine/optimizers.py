"""Optimizers with Keras (TF 2.1) semantics over a flat parameter arena.

* ``RMSprop`` — reference optimizer everywhere (``dist_model_tf_vgg.py:130,153``,
  ``fed_model.py:126,208``, ``secure_fed_model.py:96``): ``ms <- rho*ms + (1-rho)*g^2;
  w <- w - lr*g/(sqrt(ms)+eps)``, rho=0.9, eps=1e-7, ms0=0.  With momentum>0
  the TF ``ApplyRMSProp`` form ``mom <- m*mom + lr*g/sqrt(ms+eps); w -= mom`` is used.
* ``AdamW`` — Keras AdamW (decoupled weight decay, clipping by the global norm) with 32-bit or 8-bit
  moments.
* ``SGD`` — TFF's server optimizer (lr=1.0) for FedAvg.

On a GPU arena the update is ONE fused HIP kernel (``ops.optim``); on CPU the same math runs as
vectorised torch ops.  A fresh optimizer (``compile``) means fresh slot state, as in Keras.
"""
from __future__ import annotations

from typing import Optional

import torch


class Optimizer:
    name = "optimizer"

    def __init__(self, learning_rate: float):
        self.learning_rate = float(learning_rate)
        self.iterations = 0
        self._arena = None

    def bind(self, arena) -> None:
        self._arena = arena
        self._build_slots(arena)

    def _build_slots(self, arena):
        pass

    def step(self, arena=None, lr: Optional[float] = None, grad_scale: float = 1.0) -> None:
        raise NotImplementedError

    def get_config(self):
        return {"name": self.name, "learning_rate": self.learning_rate}

    # non-finite guard (SURVEY §5 failure detection): skip the whole update when any (reduced)
    # gradient is inf/nan; the fused backend does the same check on the device
    skip_nonfinite = False
    skipped = 0

    def _should_skip(self, arena) -> bool:
        if self.skip_nonfinite and not bool(torch.isfinite(arena.grad).all()):
            self.skipped += 1
            return True
        return False

    @property
    def native_step(self) -> bool:
        """Whether the fused program carries the update as a plan op (else it is a host call)."""
        return False

    def state_tensors(self):
        return {}

    def load_slots(self, slots) -> None:
        """Takes the slot tensors of a checkpoint (those that this optimizer has, in this shape)."""
        for k, v in slots.items():
            cur = self.state_tensors().get(k)
            if cur is not None and cur.shape == v.shape:
                cur.copy_(v.to(cur.device))

    def reset_state(self) -> None:
        """Zero every slot IN PLACE (pointers captured by HIP graphs stay valid)."""
        with torch.no_grad():
            for t in self.state_tensors().values():
                if t is not None:
                    t.zero_()
        self.iterations = 0


class RMSprop(Optimizer):
    name = "RMSprop"

    def __init__(self, learning_rate: float = 0.001, rho: float = 0.9, momentum: float = 0.0,
                 epsilon: float = 1e-7, centered: bool = False, lr: Optional[float] = None):
        super().__init__(lr if lr is not None else learning_rate)  # TF2.1 accepted lr=
        self.rho = float(rho)
        self.momentum = float(momentum)
        self.epsilon = float(epsilon)
        self.centered = bool(centered)
        self.ms = self.mom = self.mg = None

    def _build_slots(self, arena):
        self.ms = torch.zeros_like(arena.data)
        self.mom = torch.zeros_like(arena.data) if self.momentum > 0 else None
        self.mg = torch.zeros_like(arena.data) if self.centered else None

    def step(self, arena=None, lr=None, grad_scale: float = 1.0):
        arena = arena or self._arena
        if self._should_skip(arena):
            return
        lr = self.learning_rate if lr is None else lr
        w, g = arena.data, arena.grad
        if w.is_cuda and self.momentum == 0 and not self.centered:
            from ..ops import optim as optim_ops
            optim_ops.rmsprop_(w, g, self.ms, lr, self.rho, self.epsilon, grad_scale)
        else:
            gs = g * grad_scale if grad_scale != 1.0 else g
            self.ms.mul_(self.rho).addcmul_(gs, gs, value=1.0 - self.rho)
            denom = self.ms
            if self.centered:
                self.mg.mul_(self.rho).add_(gs, alpha=1.0 - self.rho)
                denom = self.ms - self.mg * self.mg
            if self.momentum > 0:
                self.mom.mul_(self.momentum).add_(lr * gs / torch.sqrt(denom + self.epsilon))
                w.sub_(self.mom)
            else:
                w.sub_(lr * gs / (torch.sqrt(denom) + self.epsilon))
        self.iterations += 1

    @property
    def native_step(self) -> bool:
        return self.momentum == 0 and not self.centered

    def get_config(self):
        return {"name": self.name, "learning_rate": self.learning_rate, "rho": self.rho,
                "momentum": self.momentum, "epsilon": self.epsilon, "centered": self.centered}

    def state_tensors(self):
        out = {"ms": self.ms}
        if self.mom is not None:
            out["mom"] = self.mom
        if self.mg is not None:
            out["mg"] = self.mg
        return out


class AdamW(Optimizer):
    """Keras AdamW: ``m <- b1*m + (1-b1)*g; v <- b2*v + (1-b2)*g^2;
    w <- w - lr*weight_decay*w - lr*sqrt(1-b2^t)/(1-b1^t) * m/(sqrt(v)+eps)``.

    ``global_clipnorm``: gradients are scaled down to that global norm first.  ``decay``: "all" weights
    decay, or only the "kernels" (tensors with more than one axis: no biases, no BatchNorm weights).
    ``state_bits``: 32 keeps fp32 moments (8 bytes a weight), 8 their codes (2.03 bytes; blocks of 64
    neighbouring weights share a scale, csrc/kernels/adamw.hip).  The step counter is part of the state, on
    the device.  The CPU's moments and codes are the GPU's bits (of clipped steps as long as the norm, whose
    sums have another order, rounds to the same float)."""

    name = "AdamW"

    def __init__(self, learning_rate: float = 0.001, weight_decay: float = 0.004, beta_1: float = 0.9,
                 beta_2: float = 0.999, epsilon: float = 1e-7, global_clipnorm: Optional[float] = None,
                 decay: str = "all", state_bits: int = 32, lr: Optional[float] = None):
        super().__init__(lr if lr is not None else learning_rate)
        if decay not in ("all", "kernels"):
            raise ValueError(f"decay has to be 'all' or 'kernels', not {decay!r}")
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW states have 8 or 32 bits, not {state_bits}")
        self.weight_decay = float(weight_decay)
        self.beta_1, self.beta_2, self.epsilon = float(beta_1), float(beta_2), float(epsilon)
        self.global_clipnorm = None if global_clipnorm is None else float(global_clipnorm)
        self.decay, self.state_bits = decay, int(state_bits)
        from ..ops.optim import check_adamw
        check_adamw(self.learning_rate, self.beta_1, self.beta_2, self.epsilon, self.weight_decay, self.clip_norm)
        self.table = self.state = None  # of a GPU arena (ops.optim)
        self.m = self.v = self.scales = self.steps = None

    @property
    def clip_norm(self) -> float:
        """As ops.optim takes it: 0 is no clipping."""
        return self.global_clipnorm or 0.0

    @property
    def native_step(self) -> bool:
        return True

    def _decay_runs(self, arena):
        """[(start, end, decays)]: the arena in stretches of whole slots with the same flag."""
        runs = []
        ends = [s.offset for s in arena.slots[1:]] + [arena.numel]
        for p, s, end in zip(arena.params, arena.slots, ends):
            flag = self.decay == "all" or p.dim() > 1
            if runs and runs[-1][2] == flag:
                runs[-1][1] = end
            else:
                runs.append([s.offset, end, flag])
        return runs or [[0, arena.numel, False]]

    def _build_slots(self, arena):
        runs = self._decay_runs(arena)
        if arena.data.is_cuda:
            from ..ops import optim as optim_ops
            # stretches are multiples of 64 long, so a place in the state is a place in the arena
            self.table = optim_ops.TensorTable([arena.grad[a:b] for a, b, _ in runs],
                                               [arena.data[a:b] for a, b, _ in runs], decay=[d for *_, d in runs])
            self.state = optim_ops.AdamWState(self.table, self.state_bits)
            self.m, self.v, self.scales, self.steps = self.state.m, self.state.v, self.state.scales, self.state.step
            return
        self.table = self.state = None
        dtype = torch.uint8 if self.state_bits == 8 else torch.float32
        self.m, self.v = torch.zeros_like(arena.data, dtype=dtype), torch.zeros_like(arena.data, dtype=dtype)
        self.scales = torch.zeros(arena.numel // 64, 2, dtype=torch.uint8) if self.state_bits == 8 else None
        self.steps = torch.zeros(1024, dtype=torch.int32)  # as many words as the GPU's state has
        self._mask = torch.cat([torch.full((b - a,), float(d)) for a, b, d in runs])

    def step(self, arena=None, lr=None, grad_scale: float = 1.0):
        arena = arena or self._arena
        if arena is not self._arena:
            raise ValueError("AdamW steps the arena that it is bound to")
        if self._should_skip(arena):
            return
        lr = self.learning_rate if lr is None else lr
        if self.state is not None:
            from ..ops import optim as optim_ops
            optim_ops.adamw_(self.table, self.state, lr, self.beta_1, self.beta_2, self.epsilon, self.weight_decay,
                             grad_scale, self.clip_norm)
        else:
            self._cpu_step(arena, lr, grad_scale)
        self.iterations += 1

    def _cpu_step(self, arena, lr, grad_scale):
        from ..ops import moments8
        g = arena.grad * grad_scale
        if self.clip_norm:
            norm = arena.grad.double().square().sum().sqrt().float() * abs(grad_scale)
            if not bool(norm <= self.clip_norm):
                # a quotient of two tensors: of a number and a tensor torch makes a reciprocal and a product
                g = g * (torch.full_like(norm, self.clip_norm) / norm if bool(torch.isfinite(norm)) else float("nan"))
        m, v = self.moments()
        # each product and sum rounded by itself, as the kernel does: the same bits, the same codes
        m = self.beta_1 * m + (1.0 - self.beta_1) * g
        v = self.beta_2 * v + (1.0 - self.beta_2) * (g * g)
        self.steps += 1
        t = int(self.steps[0])
        alpha = lr * (1.0 - self.beta_2 ** t) ** 0.5 / (1.0 - self.beta_1 ** t)
        root = v.sqrt()
        w = arena.data
        w.sub_(lr * self.weight_decay * self._mask * w + alpha * (m / (root + self.epsilon)))
        if self.state_bits == 32:
            self.m.copy_(m)
            self.v.copy_(v)
        else:
            low, high = moments8.dither(m.numel(), t)
            self.m[:], self.scales[:, 0] = moments8.encode(m, moments8.M_BITS, low)
            self.v[:], self.scales[:, 1] = moments8.encode(root, moments8.ROOT_BITS, high)

    def moments(self):
        """First and second moments in fp32, by place in the arena (of a 32-bit state its own tensors)."""
        if self.state is not None:
            return self.state.moments()
        return _moment_values({"m": self.m, "v": self.v, "scales": self.scales})

    def state_tensors(self):
        if self.m is None:
            return {}
        out = {"m": self.m, "v": self.v, "step": self.steps}
        if self.scales is not None:
            out["scales"] = self.scales
        return out

    def load_slots(self, slots) -> None:
        """A checkpoint's moments, of either width."""
        if self.m is None or "m" not in slots or slots["m"].shape != self.m.shape:
            return
        if slots["m"].dtype == self.m.dtype:
            super().load_slots(slots)
            return
        m, v = (t.to(self.m.device) for t in _moment_values(slots))
        if self.state is not None:
            self.state.load_moments(m, v)
        elif self.state_bits == 32:
            self.m.copy_(m)
            self.v.copy_(v)
        else:
            from ..ops import moments8
            self.m[:], self.scales[:, 0] = moments8.encode(m, moments8.M_BITS)
            self.v[:], self.scales[:, 1] = moments8.encode(v.sqrt(), moments8.ROOT_BITS)
        self.steps.fill_(int(slots["step"][0]))

    def get_config(self):
        return {"name": self.name, "learning_rate": self.learning_rate, "weight_decay": self.weight_decay,
                "beta_1": self.beta_1, "beta_2": self.beta_2, "epsilon": self.epsilon,
                "global_clipnorm": self.global_clipnorm, "decay": self.decay, "state_bits": self.state_bits}


def _moment_values(slots):
    """(m, v) in fp32 of AdamW slot tensors of either width."""
    if slots["m"].dtype != torch.uint8:
        return slots["m"], slots["v"]
    from ..ops import moments8
    root = moments8.decode(slots["v"], slots["scales"][:, 1], moments8.ROOT_BITS)
    return moments8.decode(slots["m"], slots["scales"][:, 0], moments8.M_BITS), root * root


class SGD(Optimizer):
    name = "SGD"

    def __init__(self, learning_rate: float = 0.01, momentum: float = 0.0, lr=None):
        super().__init__(lr if lr is not None else learning_rate)
        self.momentum = float(momentum)
        self.buf = None

    def _build_slots(self, arena):
        self.buf = torch.zeros_like(arena.data) if self.momentum > 0 else None

    def step(self, arena=None, lr=None, grad_scale: float = 1.0):
        arena = arena or self._arena
        if self._should_skip(arena):
            return
        lr = self.learning_rate if lr is None else lr
        g = arena.grad * grad_scale if grad_scale != 1.0 else arena.grad
        if self.buf is not None:
            self.buf.mul_(self.momentum).add_(g)
            g = self.buf
        arena.data.sub_(lr * g)
        self.iterations += 1

    def state_tensors(self):
        return {"buf": self.buf} if self.buf is not None else {}


def get(identifier) -> Optimizer:
    if isinstance(identifier, Optimizer):
        return identifier
    name = str(identifier).lower()
    if name == "rmsprop":
        return RMSprop()
    if name == "adamw":
        return AdamW()
    if name == "sgd":
        return SGD()
    raise ValueError(f"unknown optimizer {identifier!r}")
