"""AdamW for what Muon does not take: embeddings, heads, gains, biases (libmuon_amd ``muon_adamw``),
with the moments in fp32 or in fp8. The reference hands such groups to torch's own adam, as
``Muon``'s "adamw" groups do here; these optimizers have no counterpart in it.
"""

from __future__ import annotations

import torch
from torch import Tensor

from muonium_amd import _lib

from .lp_state import OptimStateFp8
from .optim import _share_memory

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _dense_like(t: Tensor, p: Tensor) -> Tensor:
    """t with its values in p's order (p is dense)."""
    if t.stride() == p.stride() or p.numel() <= 1:
        return t
    return torch.empty_like(p, dtype=t.dtype).copy_(t)


def _is_dense(p: Tensor) -> bool:
    return torch.ops.aten.is_non_overlapping_and_dense.default(p)


def _capturing(p: Tensor) -> bool:
    return (p.is_cuda and not torch.compiler.is_compiling()
            and torch.cuda.is_current_stream_capturing())


def _check_not_captured(p: Tensor, what: str) -> None:
    """What a captured step makes is made anew by every replay: state has to be there before."""
    if _capturing(p):
        raise RuntimeError(f"AdamW: {what} while a graph is captured; take a step before")


class AdamW(torch.optim.Optimizer):
    """AdamW with fp32 moments: per value, with t the parameter's step, ::

        m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
        p = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    in fp32 whatever the parameter's type, which it is rounded to once. All tensors of a device and
    type are stepped together, in two launches for up to 48 of them and one more for every 48 others.

    Args:
        params: parameters or groups of them (keys ``lr``, ``wd``, ``betas``, ``eps``, ``maximize``);
            fp32, bf16 or fp16 on HIP devices, of any layout.
        lr, wd, betas, eps, maximize: as for :class:`Muon`'s "adamw" groups, whose defaults these are.

    The state of a parameter is ``step`` (an fp32 scalar on its device), ``exp_avg`` and ``exp_avg_sq``
    (fp32, also for 16-bit parameters). A step can be captured in a HIP graph once its state
    exists (it is refused before): it counts on in every replay, with the ``lr`` and the other
    numbers that it was captured with. Parameters that share memory are stepped one after the other."""

    _moments = ("exp_avg", "exp_avg_sq")

    def __init__(
        self,
        params,
        lr: float = 1e-3,
        wd: float = 0.1,
        betas: tuple[float, float] = (0.9, 0.95),
        eps: float = 1e-8,
        maximize: bool = False,
    ):
        super().__init__(params, {"lr": lr, "wd": wd, "betas": tuple(betas), "eps": eps,
                                  "maximize": maximize})

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        problem = None
        if not 0.0 <= float(group["lr"]):
            problem = f"Invalid learning rate: {group['lr']}"
        elif not 0.0 <= group["eps"]:
            problem = f"Invalid epsilon value: {group['eps']}"
        elif not 0.0 <= group["wd"]:
            problem = f"Invalid weight decay: {group['wd']}"
        else:
            for i in range(2):
                if not 0.0 <= group["betas"][i] < 1.0:
                    problem = f"Invalid beta parameter at index {i}: {group['betas'][i]}"
        if problem is not None:
            del self.param_groups[-1]
            raise ValueError(problem)

    # -- state ------------------------------------------------------------------------

    def _block(self, p: Tensor) -> int:
        """Values that share a scale in p's moments; 0 for moments in fp32."""
        return 0

    def _new_moment(self, p: Tensor, block: int):
        if block:
            return OptimStateFp8.zeros(p.shape, block, p.device)
        return torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)

    def _init_state(self, p: Tensor) -> dict:
        state = self.state[p]
        if len(state) == 0:
            _check_not_captured(p, "a parameter has no state")
            block = self._block(p)
            state["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
            for name in self._moments if not block else AdamWFp8._quantized:
                state[name] = self._new_moment(p, block)
        return state

    def load_state_dict(self, state_dict: dict) -> None:
        """torch's own loading gives a parameter's floating-point state the parameter's type; the
        moments and the step stay fp32, on the parameter's device."""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        for group, old in zip(self.param_groups, state_dict["param_groups"]):
            for p, key in zip(group["params"], old["params"]):
                for name, value in saved.get(key, {}).items():
                    if isinstance(value, OptimStateFp8):
                        self.state[p][name] = value.to(p.device)
                    elif name == "step" or name in self._moments:
                        self.state[p][name] = torch.as_tensor(value).to(p.device, torch.float32)

    # -- the step ---------------------------------------------------------------------

    def _collect(self, params: list[Tensor]) -> dict:
        """Lists of what one call takes, by device, type and block."""
        calls: dict[tuple, tuple[list, ...]] = {}
        for p in params:
            grad = p.grad
            if grad is None:
                continue
            if grad.layout != torch.strided:
                raise RuntimeError(f"{type(self).__name__} does not support sparse gradients")
            if p.dtype not in _FLOATS:
                raise TypeError(f"parameters are fp32, bf16 or fp16; got {p.dtype}")
            state = self._init_state(p)
            m = state["exp_avg"]
            quantized = isinstance(m, OptimStateFp8)
            block = m.block_size if quantized else 0
            call = calls.setdefault((p.device, p.dtype, block), ([], [], [], [], [], [], [], []))
            # quantized blocks run along a contiguous tensor's values, other moments lie like their
            # parameter; what does not is stepped in a copy
            here = p.detach()
            if not (here.is_contiguous() if quantized else _is_dense(here)):
                here = here.contiguous()
                call[7].append((p, here))
            call[0].append(here)
            call[1].append(_dense_like(grad.detach(), here))
            if quantized:
                v = state["exp_avg_sq_root"]
                for where, t in ((2, m.codes), (3, v.codes), (4, m.scale), (5, v.scale)):
                    call[where].append(t)
            else:
                for where, name in ((2, "exp_avg"), (3, "exp_avg_sq")):
                    if (laid := _dense_like(state[name], here)) is not state[name]:
                        _check_not_captured(p, "a moment is laid out unlike its parameter")
                        state[name] = laid
                    call[where].append(laid)
            if state["step"].device != p.device:
                _check_not_captured(p, "a parameter's step is on another device")
                state["step"] = state["step"].to(p.device)
            call[6].append(state["step"])
        return calls

    @torch.no_grad()
    def step(self, closure=None):
        """One step over every group; returns the closure's loss."""
        from muonium_amd import _row_ops

        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            beta1, beta2 = group["betas"]
            numbers = (float(group["lr"]), beta1, beta2, group["eps"], float(group["wd"]),
                       group["maximize"])
            params = group["params"]
            if (_row_ops.module is not None and not torch.compiler.is_compiling()
                    and params and params[0].is_cuda):
                # plain parameters with fp32 moments are walked in C++; what it leaves is walked here
                _row_ops.check_device(params[0].device)
                left = _row_ops.module.adamw_step(params, self.state, *numbers)
                params = params if left is None else left
            for (device, _, block), call in self._collect(params).items():
                _row_ops.check_device(device)
                lists, copies = call[:7], call[7]
                if len(lists[0]) > 1 and (copies or torch.compiler.is_compiling()
                                          or _share_memory(lists[0])):
                    # in order: each sees what the ones before it left
                    for i, here in enumerate(lists[0]):
                        own = [p for p, copy in copies if copy is here]
                        for p in own:
                            here.copy_(p)
                        _row_ops.adamw_(*([x[i]] if x else [] for x in lists), block, *numbers)
                        for p in own:
                            p.copy_(here)
                else:
                    _row_ops.adamw_(*lists, block, *numbers)
                    for p, copy in copies:
                        p.copy_(copy)
        return loss


class AdamWFp8(AdamW):
    """AdamW with the moments in 8 bits: float8_e4m3fn codes, with one fp32 scale for each block of
    ``block_size`` consecutive values (:class:`OptimStateFp8`, the largest value of a block at 448).

    The state is ``step``, ``exp_avg`` and ``exp_avg_sq_root``, the second moment's root, which spans half the
    binades that v does. A root that is too small for a code beside its block's largest has the least one
    where its mean has a code, so that no step is m / eps. Without a gradient, a mean decays to 0.
    Codes are the nearest ones up to betas of 0.9375 (excluded) and 0.95, beyond which the moments would stay
    where they are: they are rounded at random there, by the step and the value's place, so that a step
    gives the same bits again and a moment follows on the average (a root by about 10 to 50% around
    its value at 0.99 and 0.999). With the nearest codes a block's roots follow as its scale moves: beside
    a largest value whose gradient never varies, small ones that do not vary either keep a root that
    is too large, and are stepped too little.
    Parameters of fewer than 4096 values, or not a multiple of ``block_size`` (``MuonLP``'s rule), have
    fp32 moments as in :class:`AdamW`.

    Args:
        block_size: a power of two from 64 to 2048.
        others: as for :class:`AdamW`."""

    _quantized = ("exp_avg", "exp_avg_sq_root")

    def __init__(
        self,
        params,
        lr: float = 1e-3,
        wd: float = 0.1,
        betas: tuple[float, float] = (0.9, 0.95),
        eps: float = 1e-8,
        maximize: bool = False,
        block_size: int = 256,
    ):
        if block_size not in (64, 128, 256, 512, 1024, 2048):
            raise ValueError(f"block_size is a power of two from 64 to 2048; got {block_size}")
        self.block_size = block_size
        super().__init__(params, lr, wd, betas, eps, maximize)

    def __getstate__(self) -> dict:
        # torch's holds the groups and the state alone
        return {**super().__getstate__(), "block_size": self.block_size}

    def __setstate__(self, state: dict) -> None:
        super().__setstate__({"block_size": 256, **state})

    def _block(self, p: Tensor) -> int:
        return self.block_size if p.numel() >= 4096 and p.numel() % self.block_size == 0 else 0
