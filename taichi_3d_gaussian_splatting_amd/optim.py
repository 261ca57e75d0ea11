"""Adam for the trainer's parameter tensors on the HIP device.

Same update rule, hyper-parameter names, ``param_groups`` and ``state_dict`` layout (``step``, ``exp_avg``,
``exp_avg_sq``) as ``torch.optim.Adam`` without weight decay / amsgrad -- what the reference instantiates at
GaussianPointTrainer.py:126-129 -- so learning-rate schedulers and checkpoints work unchanged.  The step itself is one
streaming HIP kernel per tensor (csrc/gs_optim.hip); there is no CPU path.

``AdamW`` (decoupled weight decay) steps many tensors in one launch, with moments in 32 or in 8 bits, clips by the global
norm of the gradients on the way and steps 16-bit parameters through a float32 master copy (csrc/gs_adamw.hip).  Its parts
are functions on lists of tensors: ``adamw_step_``, ``grad_norm``, ``read_moments``, ``new_moments``.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import call, check, current_stream, ptr


class Adam(torch.optim.Optimizer):
    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8):
        if lr < 0 or eps < 0 or not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("invalid Adam hyper-parameters")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps))
        self._scale_regulariser = {}   # param -> (weight, point_invalid_mask)
        self._row_mask = {}            # param -> point_invalid_mask: rows of invalid points are skipped

    def set_row_mask(self, param: torch.Tensor, point_invalid_mask: torch.Tensor) -> None:
        """``param`` is a fixed-capacity [N,3] or [N,56] tensor with one row per point and ``point_invalid_mask`` (int8 [N],
        the live tensor -- it is read at every step) marks the rows without a point: those rows are not touched by the
        step.  Their gradient is zero, so ``torch.optim.Adam`` would only decay their moments and move parameters that
        are overwritten before they are read again; the decay is applied lazily when a row comes back to life
        (``state["last_step"]``), so a row's moments are what ``torch.optim.Adam`` would hold.  With the reference's
        capacity of 10x the initial points (config/tat_truck_every_8_test.yaml:20) most rows are free for most of a
        run."""
        if param.dim() != 2 or param.shape[1] not in (3, 56) or point_invalid_mask.shape != (param.shape[0],):
            raise ValueError("set_row_mask: [N,3] or [N,56] parameter and an [N] mask")
        if point_invalid_mask.dtype != torch.int8:
            raise TypeError("point_invalid_mask must be int8")
        self._row_mask[param] = point_invalid_mask

    def set_scale_regulariser(self, features: torch.Tensor, weight: float, point_invalid_mask: torch.Tensor,
                              local_share=None) -> None:
        """Fuse the gradient of ``weight * mean_live ||exp(features[:, 4:7])||`` (the trainer's scale regulariser,
        LOS:42-54) into the step of the [N,56] parameter ``features``: it is added to the incoming gradient inside the
        Adam kernel (from the pre-step parameters), so neither autograd nor a separate pass has to produce it.
        ``weight = 0`` switches it off.

        ``local_share`` (owner-sharded Gaussians: this tensor holds only the rank's block): a zero-argument callable
        that returns n_live(this block) / n_live(all ranks).  The kernel divides by the live count it finds in the tensor
        it is given; the reference's term is a mean over ALL live Gaussians (LOS:42-54), so the weight handed to the
        kernel is ``weight * local_share()`` -- the same per-point gradient as an un-sharded run."""
        if features.dim() != 2 or features.shape[1] != 56:
            raise ValueError("the scale regulariser applies to the [N,56] feature matrix")
        if weight:
            self._scale_regulariser[features] = (float(weight), point_invalid_mask, local_share)
        else:
            self._scale_regulariser.pop(features, None)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            beta1, beta2 = group["betas"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not (p.is_cuda and p.dtype == torch.float32 and p.is_contiguous()):
                    raise RuntimeError("optim.Adam needs contiguous float32 parameters on the HIP device")
                grad = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
                state = self.state[p]
                if not state:
                    state["step"] = 0
                    state["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                    state["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                state["step"] = int(state["step"]) + 1
                reg = self._scale_regulariser.get(p)
                mask = self._row_mask.get(p)
                if mask is not None:
                    if reg is not None and reg[1] is not mask:
                        raise RuntimeError("set_row_mask and set_scale_regulariser were given different masks")
                    if "last_step" not in state:
                        # moments restored from a state_dict written without row masks (or by torch.optim.Adam) are
                        # current as of the previous step: no lazy decay is owed for them
                        state["last_step"] = torch.full((p.shape[0],), int(state["step"]) - 1, dtype=torch.int32,
                                                        device=p.device)
                    weight = (reg[0] * (float(reg[2]()) if reg[2] is not None else 1.0)) if reg is not None else 0.0
                    ws = torch.empty(256, dtype=torch.int32, device=p.device) if weight else None
                    call("gs_adam_step_rows", ptr(p), ptr(grad), ptr(state["exp_avg"]), ptr(state["exp_avg_sq"]),
                         p.shape[0], p.shape[1], float(group["lr"]), float(beta1), float(beta2), float(group["eps"]),
                         state["step"], ptr(mask), ptr(state["last_step"]), float(weight), ptr(ws),
                         current_stream(p.device))
                    continue
                if reg is not None:
                    weight, mask = reg[0] * (float(reg[2]()) if reg[2] is not None else 1.0), reg[1]
                    ws = torch.empty(256, dtype=torch.int32, device=p.device)
                    call("gs_adam_step_features", ptr(p), ptr(grad), ptr(state["exp_avg"]), ptr(state["exp_avg_sq"]),
                         p.shape[0], float(group["lr"]), float(beta1), float(beta2), float(group["eps"]), state["step"],
                         ptr(mask), weight, ptr(ws), current_stream(p.device))
                    continue
                call("gs_adam_step", ptr(p), ptr(grad), ptr(state["exp_avg"]), ptr(state["exp_avg_sq"]), p.numel(),
                     float(group["lr"]), float(beta1), float(beta2), float(group["eps"]), state["step"],
                     current_stream(p.device))
        return loss


# ---------------------------------------------------------------------------------------------- AdamW over many tensors
MOMENT_BLOCK = 64        # elements that share the exponents of their 8-bit moments (a row of at most 64, where there are rows)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # GS_DTYPE_*
Scalar = Union[float, torch.Tensor]


def _row_length(shape) -> int:
    """Columns of a two-dimensional tensor whose rows are blocks (1..64 columns), else 0: blocks of 64 elements."""
    return int(shape[1]) if len(shape) == 2 and 1 <= shape[1] <= MOMENT_BLOCK else 0


def _num_blocks(shape) -> int:
    row = _row_length(shape)
    return int(shape[0]) if row else -(-int(torch.Size(shape).numel()) // MOMENT_BLOCK)


def new_moments(param: torch.Tensor, bits: int = 32) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """``(exp_avg, exp_avg_sq, exponents)`` of zeros for ``param``: float32 tensors and None with 32 bits; with 8 bits uint8
    tensors of codes in the parameter's shape and uint8 ``[blocks, 2]`` exponents (of the first and the second moment).  A
    block is a row of a two-dimensional parameter with at most 64 columns, else 64 consecutive elements."""
    if bits == 32:
        zeros = [torch.zeros(param.shape, dtype=torch.float32, device=param.device) for _ in range(2)]
        return zeros[0], zeros[1], None
    if bits != 8:
        raise ValueError(f"moments in 8 or 32 bits, not {bits}")
    codes = [torch.zeros(param.shape, dtype=torch.uint8, device=param.device) for _ in range(2)]
    return codes[0], codes[1], torch.zeros(_num_blocks(param.shape), 2, dtype=torch.uint8, device=param.device)


def _on(device_index: int):
    """The device made current for a call's launches, if it is not."""
    return contextlib.nullcontext() if torch.cuda.current_device() == device_index else torch.cuda.device(device_index)


def _stream(device_index: int) -> int:
    """Handle of the current stream (``_lib.current_stream`` without the stream object: a small step is 7 us in all)."""
    return torch._C._cuda_getCurrentRawStream(device_index)


def _capturing(device_index: int) -> bool:
    """Whether the device's current stream is being captured into a graph (a host tensor's, -1, never is)."""
    if device_index < 0:
        return False
    with _on(device_index):
        return torch.cuda.is_current_stream_capturing()


def _norm_of(host, collected, grads, masks, max_norm: float, each: bool, group=None) -> torch.Tensor:
    """[norm, clip, each ...] of collected gradients, on their device's current stream."""
    index = collected[4]
    device, n = torch.device("cuda", index), len(collected[1]) // 8
    words = (2 + (n if each else 0) + 1) // 2 * 2       # behind them: the sum of squares (double), the library's workspace
    out = torch.empty(words + 2 + (_lib.load().gs_grad_norm_workspace_bytes(n) + 3) // 4, dtype=torch.float32, device=device)
    floats = out.data_ptr()
    sq_sum = floats + 4 * words
    with _on(index):
        stream = _stream(index)
        check(host.norm(grads, masks, collected, max_norm, sq_sum, floats, floats + 4, floats + 8 if each else 0, sq_sum + 8, stream),
              "gs_grad_norm")
        if group is not None:
            _sum_over_ranks(out[words:words + 2].view(torch.float64), group)
            call("gs_clip_coefficient", sq_sum, max_norm, floats, floats + 4, stream)
    return out


def _sum_over_ranks(value: torch.Tensor, group=None) -> None:
    import torch.distributed as dist
    if dist.get_backend(group) == "nccl":
        dist.all_reduce(value, group=group)
        return
    host = value.cpu()          # other back ends get host memory
    dist.all_reduce(host, group=group)
    value.copy_(host)


def grad_norm(grads: Sequence[torch.Tensor], row_masks: Optional[Sequence[Optional[torch.Tensor]]] = None, *,
              per_tensor: bool = False):
    """2-norm of all ``grads`` together (float32 scalar on their device, no host wait); with ``per_tensor`` also the norms of
    each (float32 ``[len(grads)]``).  float32, bfloat16 and float16 tensors may be mixed; squares are added up in double
    precision in a fixed order, so equal inputs give equal bits.  ``row_masks``: int8 ``[N]`` (or None) for each tensor; rows
    ``[N, 1..64]`` with a mask other than 0 do not count, whatever they hold.  An infinite or NaN gradient shows in the norm."""
    if len(grads) == 0:
        raise ValueError("grad_norm: no gradients")
    host = _lib.host()
    collected = host.collect(("grads", grads, host.GRADS), ("row_masks", row_masks, host.MASK))
    out = _norm_of(host, collected, *collected[0], 0.0, per_tensor)
    return (out[0], out[2:2 + len(grads)]) if per_tensor else out[0]


def adamw_step_(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
                exp_avg_sqs: Sequence[torch.Tensor], *, step: Union[int, torch.Tensor, Sequence[Union[int, torch.Tensor]]],
                lr: Union[Scalar, Sequence[Scalar]] = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                weight_decay: Union[float, Sequence[float]] = 1e-2,
                exponents: Optional[Sequence[torch.Tensor]] = None,
                masters: Optional[Sequence[Optional[torch.Tensor]]] = None,
                row_masks: Optional[Sequence[Optional[torch.Tensor]]] = None,
                last_steps: Optional[Sequence[Optional[torch.Tensor]]] = None,
                max_grad_norm: Optional[float] = None, norm_group=None, grad_scale: Optional[torch.Tensor] = None,
                seed: int = 0, tensor_ids: Optional[Sequence[int]] = None) -> Optional[torch.Tensor]:
    """One AdamW step of many tensors in place, as few launches as their types need.  With ``t`` a tensor's step::

        g = grad * clip;  m += (1 - b1) (g - m);  v = b2 v + (1 - b2) g g
        p = p (1 - lr weight_decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    * ``params`` / ``grads``: contiguous tensors on one HIP device, each pair of one type: float32, bfloat16 or float16.
    * ``exp_avgs`` / ``exp_avg_sqs`` / ``exponents``: as ``new_moments`` makes them -- float32 without exponents, or uint8 codes
      with them.  8-bit moments are rounded at random so that their mean is kept (a code is 1/16 to 1/8 of its value, far more
      than a step moves the second moment): the bits are a hash of ``seed``, the tensor's id (``tensor_ids``, else its place in
      the list), its step and the element, so equal calls give equal results.  A block in which a moment is infinite or NaN
      becomes NaN as a whole; finite ones at the end of float32's range (over 2.97e38) are held as the largest code.
    * ``masters``: float32 copies (or None) of 16-bit parameters; the step runs on the copy and the parameter receives its
      rounded value.  Without a copy the parameter itself is rounded to nearest, and steps below half its spacing are lost.
    * ``step``: this step's number (from 1), or a device tensor (int64, one element) that holds it when the kernels run;
      ``lr``: a number or a device tensor (float32, one element); each for all tensors or one per tensor.  While a graph is
      captured ``step`` has to be a tensor: a number would be the same at every replay.
    * ``row_masks`` / ``last_steps``: for float32 tensors ``[N, 1..64]``, int8 ``[N]`` and int32 ``[N]``: rows with a mask
      other than 0 are left as they are, and a row that missed ``d`` steps starts from ``m b1^d``, ``v b2^d``.
    * ``max_grad_norm``: gradients are scaled by ``min(1, max_grad_norm / (norm + 1e-6))`` as they are read; the norm is that of
      all gradients of the call (masked rows apart), over all ranks of ``norm_group`` where one is given (each of them calls
      with one tensor at least), and is returned as a float32 scalar on the device.  ``grads`` themselves stay as they are.  An
      infinite norm scales by 0, a NaN makes NaN of everything, as torch.nn.utils.clip_grad_norm_ does.
    * ``grad_scale``: a float32 device scalar to multiply the gradients with instead.

    Nothing waits for the device (but for a ``norm_group`` whose back end takes host memory).  Written buffers must not
    overlap anything else in the call."""
    n = len(params)
    if (row_masks is None) != (last_steps is None):
        raise ValueError("row_masks and last_steps come together")
    if max_grad_norm is not None and not max_grad_norm > 0:
        raise ValueError("max_grad_norm must be positive (None: no clipping)")
    if max_grad_norm is not None and grad_scale is not None:
        raise ValueError("max_grad_norm and grad_scale exclude each other")
    beta1, beta2 = betas
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1 and eps >= 0):
        raise ValueError("invalid AdamW hyper-parameters")
    if tensor_ids is not None and len(tensor_ids) != n:
        raise ValueError(f"tensor_ids: {len(tensor_ids)} entries for {n} tensors")
    host = _lib.host()
    moment = host.FLOAT if exponents is None else host.CODE
    collected = host.collect(("params", params, host.PARAM), ("grads", grads, host.GRAD), ("exp_avgs", exp_avgs, moment),
                             ("exp_avg_sqs", exp_avg_sqs, moment), ("exponents", exponents, host.EXPONENTS),
                             ("masters", masters, host.MASTER), ("row_masks", row_masks, host.PARAM_MASK),
                             ("last_steps", last_steps, host.STAMP))
    if n == 0:
        if max_grad_norm is not None:
            raise ValueError("the norm of no gradients")
        return None
    columns, index = collected[0], collected[4]
    if grad_scale is not None and (grad_scale.get_device() != index or grad_scale.dtype is not torch.float32 or grad_scale.numel() != 1):
        raise ValueError("grad_scale: one float32 on the parameters' device")
    numbers = host.scalars(n, step, lr, weight_decay, beta1, beta2, eps, index)
    norms, clip = None, 0
    with _on(index):
        if numbers[4] and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured step needs its step count in a device tensor: a number would be the same at every replay")
        if max_grad_norm is not None:
            norms = _norm_of(host, collected, columns[1], columns[6], float(max_grad_norm), False, norm_group)
            clip = norms.data_ptr() + 4
        elif grad_scale is not None:
            clip = grad_scale.data_ptr()
        workspace, workspace_at = None, 0
        if numbers[2] is not None or numbers[3] is not None:
            workspace = torch.empty(int(_lib.load().gs_adamw_workspace_bytes(n)), dtype=torch.uint8, device=torch.device("cuda", index))
            workspace_at = workspace.data_ptr()
        check(host.step(collected, numbers, tensor_ids, clip, seed & 0xFFFFFFFF, workspace_at, _stream(index)), "gs_adamw_step")
    return None if norms is None else norms[0]


def read_moments(exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor], exponents: Sequence[torch.Tensor], *,
                 dtype: torch.dtype = torch.float32, out: Optional[Tuple[Sequence[torch.Tensor], Sequence[torch.Tensor]]] = None
                 ) -> Tuple[Sequence[torch.Tensor], Sequence[torch.Tensor]]:
    """The values that 8-bit moments stand for, as two lists of ``dtype`` tensors (float32 or bfloat16: both hold every value
    exactly) or written to ``out``."""
    n = len(exp_avgs)
    host = _lib.host()
    inputs = ("exp_avgs", exp_avgs, host.CODE), ("exp_avg_sqs", exp_avg_sqs, host.CODE), ("exponents", exponents, host.EXPONENTS)
    if out is None:
        if dtype not in (torch.float32, torch.bfloat16):
            raise TypeError("read_moments: float32 or bfloat16 values")
        host.collect(*inputs)
        out = tuple([torch.empty(t.shape, dtype=dtype, device=t.device) for t in exp_avgs] for _ in range(2))
    collected = host.collect(*inputs, ("out", out[0], host.VALUE), ("out", out[1], host.VALUE))
    if n == 0:
        return out
    dtype = out[0][0].dtype
    if out[1][0].dtype is not dtype:
        raise TypeError("out: both lists have one type")
    index = collected[4]
    with _on(index):
        check(host.read(collected, _DTYPES[dtype], _stream(index)), "gs_read_moments")
    return out


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW``'s rule (decoupled weight decay, no amsgrad) for float32, bfloat16 and float16 parameters on the
    HIP device, all of them in one call of ``adamw_step_``.

    * ``state_bits`` (also per group): 32 (float32 moments) or 8 (a code and a share of two exponents each: 2.03 bytes for an
      element's two moments instead of 8), see ``new_moments``; ``moments(param)`` reads either.
    * ``master_weights``: 16-bit parameters are stepped through a float32 copy (``state["master"]``, made at the first step; who
      changes such a parameter afterwards changes the copy too).
    * ``max_grad_norm``: the gradients of all groups are clipped by their global norm; ``last_grad_norm`` holds it (a device
      scalar) after a step.  ``norm_group``: a process group whose ranks hold different parameters: the norm is that of all.
    * ``capturable``: step counts live on the device, so a step can be captured into a graph and replayed; ``lr`` may then be a
      float32 device tensor.  Run one step before the capture: the state is made there.
    * ``seed``: of the rounding of 8-bit moments.

    ``param_groups`` and the state's ``step`` / ``exp_avg`` / ``exp_avg_sq`` are named as in torch; a state_dict of
    ``torch.optim.AdamW`` loads into 32-bit moments."""

    def __init__(self, params, lr: Scalar = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32, master_weights: bool = True, max_grad_norm: Optional[float] = None, norm_group=None,
                 capturable: bool = False, seed: int = 0):
        if (not isinstance(lr, torch.Tensor) and lr < 0) or eps < 0 or weight_decay < 0 or not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("invalid AdamW hyper-parameters")
        if state_bits not in (8, 32):
            raise ValueError(f"moments in 8 or 32 bits, not {state_bits}")
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError("max_grad_norm must be positive (None: no clipping)")
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("a learning rate in a tensor needs capturable=True")
        self.master_weights, self.max_grad_norm, self.norm_group = bool(master_weights), max_grad_norm, norm_group
        self.capturable, self.seed = bool(capturable), int(seed)
        self.last_grad_norm: Optional[torch.Tensor] = None
        self._row_mask = {}            # param -> point_invalid_mask
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def set_row_mask(self, param: torch.Tensor, point_invalid_mask: torch.Tensor) -> None:
        """As ``Adam.set_row_mask``, for any float32 parameter ``[N, 1..64]``: rows marked in the int8 ``[N]`` mask (the live
        tensor, read at every step) are not touched and do not count in the norm; their moments decay lazily."""
        if _row_length(param.shape) == 0 or point_invalid_mask.shape != param.shape[:1]:
            raise ValueError(f"set_row_mask: [N, 1..{MOMENT_BLOCK}] parameter and an [N] mask")
        if point_invalid_mask.dtype != torch.int8 or param.dtype != torch.float32:
            raise TypeError("set_row_mask: float32 parameter and int8 mask")
        self._row_mask[param] = point_invalid_mask

    def _new_state(self, p: torch.Tensor, group: dict) -> dict:
        m, v, exponents = new_moments(p, group["state_bits"])
        state = dict(step=torch.zeros((), dtype=torch.int64, device=p.device) if self.capturable else 0, exp_avg=m, exp_avg_sq=v)
        if exponents is not None:
            state["exponents"] = exponents
        if self.master_weights and p.dtype != torch.float32:
            state["master"] = p.detach().to(torch.float32)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = self._work()
        if not work:
            if self.max_grad_norm is not None:
                device = next(p.device for group in self.param_groups for p in group["params"])
                share = torch.zeros(1, dtype=torch.float64, device=device)
                if self.norm_group is not None:     # (the other ranks wait for this one's share)
                    _sum_over_ranks(share, self.norm_group)
                self.last_grad_norm = share.sqrt().float()[0]
            return loss
        clip = None
        if self.max_grad_norm is not None:
            if len({key[3] for key in work}) > 1:
                raise RuntimeError("max_grad_norm: all parameters belong on one device")
            clip = self._clip(list(work.values()))
        for (eight, betas, eps, _), (params, grads, states, masks, rates, decays, ids) in work.items():
            if self.capturable:
                steps = [s["step"] for s in states]
                torch._foreach_add_(steps, 1)
            else:
                steps = [s["step"] + 1 for s in states]
            masters = [s.get("master") for s in states] if self.master_weights else None
            masked = any(mask is not None for mask in masks)
            try:
                adamw_step_(params, grads, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], step=steps, lr=rates,
                            betas=betas, eps=eps, weight_decay=decays,
                            exponents=[s["exponents"] for s in states] if eight else None, masters=masters,
                            row_masks=masks if masked else None,
                            last_steps=[None if mask is None else s["last_step"] for s, mask in zip(states, masks)] if masked else None,
                            grad_scale=clip, seed=self.seed, tensor_ids=ids)
            except Exception:
                if self.capturable:         # (a refused step has not happened)
                    torch._foreach_add_(steps, -1)
                raise
            if not self.capturable:
                for state, count in zip(states, steps):
                    state["step"] = count
            if masked:                  # (without a mask no row is late any more)
                for p, state in zip(params, states):
                    if p not in self._row_mask:
                        state.pop("last_step", None)
        return loss

    def _work(self) -> dict:
        """What a step has to do, by what one call of ``adamw_step_`` shares: (8-bit moments, betas, eps, device index) -> lists of
        parameters, gradients, states, row masks, rates, decays and the parameters' places in the optimiser."""
        work, place = {}, 0
        for group in self.param_groups:
            params, first = group["params"], place
            place += len(params)
            grads = [p.grad for p in params]
            ids = list(range(first, place))
            if any(g is None for g in grads):
                kept = [i for i, g in enumerate(grads) if g is not None]
                params, grads, ids = ([column[i] for i in kept] for column in (params, grads, ids))
            states = [self.state[p] for p in params]
            masks = [self._row_mask.get(p) for p in params] if self._row_mask else [None] * len(params)
            for i, state in enumerate(states):
                if state and (masks[i] is None) != ("last_step" in state):
                    continue
                if state and masks[i] is None:
                    masks[i] = self._no_row_masked(params[i])
                else:
                    self._complete(params[i], state, masks[i], group)
            kinds = [("exponents" in s, p.get_device()) for p, s in zip(params, states)]
            for kind in sorted(set(kinds)):
                columns = params, grads, states, masks, ids
                if any(k != kind for k in kinds):
                    columns = tuple([x for x, k in zip(column, kinds) if k == kind] for column in columns)
                n = len(columns[0])
                rows = work.setdefault((kind[0], tuple(group["betas"]), group["eps"], kind[1]), tuple([] for _ in range(7)))
                for row, column in zip(rows, (*columns[:4], [group["lr"]] * n, [group["weight_decay"]] * n, columns[4])):
                    row.extend(column)
        return work

    def _complete(self, p: torch.Tensor, state: dict, mask: Optional[torch.Tensor], group: dict) -> None:
        """The state of a parameter that has none, or none for its row mask yet."""
        if not state and not p.is_cuda:
            raise RuntimeError("optim.AdamW needs parameters on the HIP device: there is no CPU path")
        if _capturing(p.get_device()):
            raise RuntimeError("run one step of AdamW before capturing one: its state is made there")
        if not state:
            state.update(self._new_state(p, group))
        if mask is not None:
            # moments from a state_dict without row masks are current as of the previous step
            state["last_step"] = torch.full((p.shape[0],), int(state["step"]), dtype=torch.int32, device=p.device)

    def _no_row_masked(self, p: torch.Tensor) -> torch.Tensor:
        """For a parameter whose state comes from steps under a row mask and that has no mask now: one that lets every row take
        this step, late ones with their decay.  The stamps end with it: the steps after it would not keep them."""
        if _capturing(p.get_device()):
            raise RuntimeError("run one step of AdamW before capturing one: rows that an earlier mask held back take it there")
        return torch.zeros(p.shape[0], dtype=torch.int8, device=p.device)

    def _clip(self, parts) -> torch.Tensor:
        """The clipping coefficient of all gradients (and ``last_grad_norm``)."""
        host = _lib.host()
        grads, masks = [g for columns in parts for g in columns[1]], [mask for columns in parts for mask in columns[3]]
        collected = host.collect(("grads", grads, host.GRADS), ("row_masks", masks, host.MASK))
        norms = _norm_of(host, collected, *collected[0], float(self.max_grad_norm), False, self.norm_group)
        self.last_grad_norm = norms[0]
        return norms[1]

    def moments(self, param: torch.Tensor, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """Copies of a parameter's first and second moment in any type, whatever they are held in (of rows that miss steps under a
        row mask: as of the last step that reached them)."""
        state = self.state.get(param)
        if not state:
            raise KeyError("the parameter has no state yet")
        if "exponents" not in state:
            return state["exp_avg"].to(dtype, copy=True), state["exp_avg_sq"].to(dtype, copy=True)
        held = [state["exp_avg"]], [state["exp_avg_sq"]], [state["exponents"]]
        (m,), (v,) = read_moments(*held, dtype=dtype if dtype == torch.bfloat16 else torch.float32)
        return m.to(dtype), v.to(dtype)

    _OPTIONS = ("master_weights", "max_grad_norm", "norm_group", "capturable", "seed", "last_grad_norm")

    def __getstate__(self) -> dict:
        places = {p: i for i, p in enumerate(p for group in self.param_groups for p in group["params"])}
        return {**super().__getstate__(), **{name: getattr(self, name) for name in self._OPTIONS},
                "row_masks": {places[i]: mask for i, mask in self._row_mask.items() if i in places}}

    def __setstate__(self, state: dict) -> None:
        state = dict(state)
        masks = state.pop("row_masks", None)
        super().__setstate__(state)
        if masks is not None:       # (a copy or an unpickled optimiser; load_state_dict brings none)
            params = [p for group in self.param_groups for p in group["params"]]
            self._row_mask = {params[i]: mask for i, mask in masks.items()}

    def load_state_dict(self, state_dict) -> None:
        """As in torch, hooks among it, but the state keeps its own types (torch would cast codes, counts and float32 moments of
        16-bit parameters to the parameter's type).  Whether moments have 8 or 32 bits is what was saved; options that a saved
        group does not name stay the group's own; amsgrad and maximize are not known here.  A state_dict that does not fit is
        refused and changes nothing."""
        params = [p for group in self.param_groups for p in group["params"]]
        states = []

        def take(_, given):         # (behind the other hooks: what they return is what is loaded)
            saved_groups = given["param_groups"]
            for group in saved_groups:
                if group.get("amsgrad") or group.get("maximize"):
                    raise ValueError("state_dict: AdamW here has neither amsgrad nor maximize")
            held = [given["state"].get(i) for group in saved_groups for i in group["params"]]
            states.extend(self._loaded(p, h) if h else None for p, h in zip(params, held))
            kept = [{name: group[name] for name in self.defaults if name in group} for group in self.param_groups]
            kept += [{}] * (len(saved_groups) - len(kept))
            return {**given, "state": {}, "param_groups": [{**own, **group} for own, group in zip(kept, saved_groups)]}

        def put(_):                 # (in front of the other hooks: they find the state)
            self.state.clear()
            self.state.update((p, state) for p, state in zip(params, states) if state is not None)
            for group in self.param_groups:
                for p in group["params"]:
                    if p in self.state:
                        group["state_bits"] = 8 if "exponents" in self.state[p] else 32
        handles = [self.register_load_state_dict_pre_hook(take), self.register_load_state_dict_post_hook(put, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for handle in handles:
                handle.remove()

    def _loaded(self, p: torch.Tensor, held: dict) -> dict:
        """A saved state as this optimiser's, on the parameter's device."""
        shapes = {"exp_avg": p.shape, "exp_avg_sq": p.shape, "master": p.shape, "exponents": (_num_blocks(p.shape), 2),
                  "last_step": p.shape[:1]}
        eight = "exponents" in held
        moment = torch.uint8 if eight else torch.float32
        types = {"exp_avg": moment, "exp_avg_sq": moment, "exponents": torch.uint8, "master": torch.float32, "last_step": torch.int32}
        if not {"step", "exp_avg", "exp_avg_sq"} <= set(held):
            raise ValueError("state_dict: no AdamW state")
        count = int(held["step"])
        state = dict(step=torch.full((), count, dtype=torch.int64, device=p.device) if self.capturable else count)
        for name, shape in shapes.items():
            if name not in held or (name == "master" and (not self.master_weights or p.dtype == torch.float32)):
                continue
            value = held[name]
            if name == "last_step" and (_row_length(p.shape) == 0 or p.dtype != torch.float32):
                raise ValueError("state_dict: last_step belongs to a float32 parameter of rows")
            if tuple(value.shape) != tuple(shape):
                raise ValueError(f"state_dict: {name} has shape {tuple(value.shape)}, not {tuple(shape)}")
            if (value.dtype == torch.uint8) != (types[name] == torch.uint8):
                raise TypeError(f"state_dict: {name} is {value.dtype}, not {types[name]}")
            state[name] = value.detach().to(device=p.device, dtype=types[name], copy=True).contiguous()
        if self.master_weights and p.dtype != torch.float32 and "master" not in state:
            state["master"] = p.detach().to(torch.float32)
        return state
