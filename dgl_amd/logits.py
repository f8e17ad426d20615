"""From logits to log-probabilities under a search's controls (include/dgl_amd.h, dgl_logits_t).

The reference turns the policy's logits into probabilities by a feasibility-masked softmax (TSP/TSPModel.py:317-337) and
hands their logarithms to Beamsearch.advance.  ``process_logits`` is that step with the controls a search may want:
penalties for actions in a row's history, biases on actions, a temperature, and blocked actions as the states' visited words
hold them."""
from __future__ import annotations

import ctypes
import struct
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._lib import ptr
from .attention import _DTYPES, _launch, _side, derivatives, no_derivatives

PerRow = Union[float, torch.Tensor]
_PACK = struct.Struct("@4iPqPq2iPqPq4P4fPqP")
assert _PACK.size == ctypes.sizeof(_lib.Logits)


@dataclass
class LogitControls:
    """What ``process_logits`` applies at every decision of a rollout (TspEngine / CvrpEngine.greedy_rollout and
    beam_rollout; the testers' ``tester_params['logit_controls']``), on top of the states' own masks.

    ``bias`` [actions] or [rows, actions]; ``temperature``; ``blocked`` int64 words [rows, n], actions never taken while the
    policy offers another one - its feasible candidates at that decision, not every node that is left: a row whose candidates
    are all blocked takes the policy's own choice; ``history`` int32 [rows, n] with ``history_len`` [rows] live entries, actions
    to penalise - for instance the first moves of solutions found earlier.

    They apply to the policy's log-probabilities, which are never positive: a repetition penalty always multiplies.  Row-wise
    controls belong to the engine's rows and stay with them.  In a beam rollout a row is a slot of its beam, which hypotheses
    enter and leave: give all slots of a beam the same."""
    bias: Optional[torch.Tensor] = None
    temperature: float = 1.0
    repetition: PerRow = 1.0
    presence: PerRow = 0.0
    frequency: PerRow = 0.0
    history: Optional[torch.Tensor] = None
    history_len: Optional[torch.Tensor] = None
    blocked: Optional[torch.Tensor] = None


def process_logits(logits: torch.Tensor, *, blocked: Optional[torch.Tensor] = None, period: Optional[int] = None,
                   bias: Optional[torch.Tensor] = None, temperature: float = 1.0, history: Optional[torch.Tensor] = None,
                   history_len: Optional[torch.Tensor] = None, repetition: PerRow = 1.0, presence: PerRow = 0.0,
                   frequency: PerRow = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(log_probs [R, A] float32, selected [R] int32) of logits [R, A] (float32, float16, bfloat16).

    Actions that occur c > 0 times in ``history`` [R, n] (its first ``history_len`` [R] entries):
    x = (x > 0 ? x / repetition : x * repetition) - presence - frequency * c.  Then x = (x + bias) / temperature, and -inf
    where bit (a mod ``period``) of ``blocked`` [R, words] is set (``period``: default A; CVRP's direct and via-depot moves
    share N + 1 bits).  log_probs is the log-softmax of what is left, ``selected`` its lowest greatest action (-1 and -inf
    throughout where all is blocked).  Penalties are numbers or float tensors [R].  For decisions: inputs that require grad are
    refused."""
    penalties = [x if isinstance(x, torch.Tensor) else None for x in (repetition, presence, frequency)]
    if derivatives(logits, bias, *penalties):
        no_derivatives("process_logits", logits=logits, bias=bias, repetition=penalties[0], presence=penalties[1],
                       frequency=penalties[2])
    if logits.dim() != 2 or logits.dtype not in _DTYPES or not logits.is_cuda:
        raise ValueError(f"logits are {tuple(logits.shape)} {logits.dtype} on {logits.device}: [rows, actions] of float32, "
                         "float16 or bfloat16 on a GPU are expected")
    R, A = logits.shape
    dev = logits.device
    if A < 1:
        raise ValueError("no actions")
    if logits.stride(1) != 1 and A > 1:
        logits = logits.contiguous()
    words = bits_stride = cols = history_stride = bias_stride = 0
    if blocked is not None:
        if blocked.dim() != 2 or blocked.shape[0] != R or blocked.dtype != torch.int64 or blocked.device != dev:
            raise ValueError(f"blocked is {tuple(blocked.shape)} {blocked.dtype}: int64 words [{R}, n] on {dev} are expected")
        words = blocked.shape[1]
        if words > 1 and blocked.stride(1) != 1:
            blocked = blocked.contiguous()
        bits_stride = blocked.stride(0)
    if bias is not None:
        bias = _side(bias, "bias", (A,) if bias.dim() == 1 else (R, A), torch.float32, dev)
        bias_stride = 0 if bias.dim() == 1 else bias.stride(0)
    if history_len is not None and history is None:
        raise ValueError("history_len without a history")
    if history is not None:
        if history.dim() != 2:
            raise ValueError(f"history has shape {tuple(history.shape)}: [{R}, n] is expected")
        history = _side(history, "history", (R, history.shape[1]), torch.int32, dev)
        history_len = _side(history_len, "history_len", (R,), torch.int32, dev)
        cols, history_stride = history.shape[1], history.stride(0)
    rows, numbers = [], []
    for name, x, t, neutral in (("repetition", repetition, penalties[0], 1.0), ("presence", presence, penalties[1], 0.0),
                                ("frequency", frequency, penalties[2], 0.0)):
        rows.append(_side(t, name, (R,), torch.float32, dev))
        numbers.append(float(x) if t is None else neutral)
    out = torch.empty((R, A), dtype=torch.float32, device=dev)
    selected = torch.empty(R, dtype=torch.int32, device=dev)
    if R == 0:
        return out, selected
    a = _lib.Logits()
    _PACK.pack_into(a, 0, _DTYPES[logits.dtype], R, A, A if period is None else int(period), logits.data_ptr(), logits.stride(0),
                    ptr(blocked), bits_stride, words, cols, ptr(bias), bias_stride, ptr(history) if cols else 0, history_stride,
                    ptr(history_len), ptr(rows[0]), ptr(rows[1]), ptr(rows[2]), *numbers, float(temperature), out.data_ptr(), A,
                    selected.data_ptr())
    lib, ref = _lib.load(), ctypes.byref(a)
    need = lib.dgl_logits_workspace_floats(ref)
    ws = torch.empty(need, dtype=torch.float32, device=dev) if need > 0 else None
    _launch(dev, lib.dgl_logits_process, ref, ptr(ws), what="dgl_logits_process")
    return out, selected
