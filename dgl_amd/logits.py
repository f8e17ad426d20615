"""From logits to log-probabilities under a search's controls (include/dgl_amd.h, dgl_logits_t).

The reference turns the policy's logits into probabilities by a feasibility-masked softmax (TSP/TSPModel.py:317-337) and
hands their logarithms to Beamsearch.advance.  ``process_logits`` is that step with the controls a search may want:
penalties for actions in a row's history, biases on actions, a temperature, and blocked actions as the states' visited words
hold them."""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._lib import check, ptr
from .attention import _DTYPES, _on, _side, _stream

PerRow = Union[float, torch.Tensor]


@dataclass
class LogitControls:
    """What ``process_logits`` applies at every decision of a rollout (TspEngine / CvrpEngine.greedy_rollout and
    beam_rollout; the testers' ``tester_params['logit_controls']``), on top of the states' own masks.

    ``bias`` [actions] or [rows, actions]; ``temperature``; ``blocked`` int64 words [rows, n], actions never taken while
    another one is left; ``history`` int32 [rows, n] with ``history_len`` [rows] live entries, actions to penalise - for
    instance the first moves of solutions found earlier."""
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
    throughout where all is blocked).  Penalties are numbers or float tensors [R]."""
    with torch.no_grad():
        if logits.dim() != 2 or logits.dtype not in _DTYPES or not logits.is_cuda:
            raise ValueError(f"logits are {tuple(logits.shape)} {logits.dtype} on {logits.device}: [rows, actions] of float32, "
                             "float16 or bfloat16 on a GPU are expected")
        R, A = logits.shape
        dev = logits.device
        if A < 1:
            raise ValueError("no actions")
        if logits.stride(1) != 1 and A > 1:
            logits = logits.contiguous()
        a = _lib.Logits()
        a.dtype, a.R, a.A, a.period = _DTYPES[logits.dtype], R, A, A if period is None else int(period)
        a.logits, a.logits_stride, a.temperature = ptr(logits), logits.stride(0), float(temperature)
        keep = []
        if blocked is not None:
            if blocked.dim() != 2 or blocked.shape[0] != R or blocked.dtype != torch.int64 or blocked.device != dev:
                raise ValueError(f"blocked is {tuple(blocked.shape)} {blocked.dtype}: int64 words [{R}, n] on {dev} are expected")
            if blocked.shape[1] > 1 and blocked.stride(1) != 1:
                blocked = blocked.contiguous()
            keep.append(blocked)
            a.blocked, a.blocked_stride, a.words = ptr(blocked), blocked.stride(0), blocked.shape[1]
        if bias is not None:
            bias = _side(bias, "bias", (A,) if bias.dim() == 1 else (R, A), torch.float32, dev)
            keep.append(bias)
            a.bias, a.bias_stride = ptr(bias), 0 if bias.dim() == 1 else bias.stride(0)
        if history_len is not None and history is None:
            raise ValueError("history_len without a history")
        if history is not None:
            if history.dim() != 2:
                raise ValueError(f"history has shape {tuple(history.shape)}: [{R}, n] is expected")
            history = _side(history, "history", (R, history.shape[1]), torch.int32, dev)
            history_len = _side(history_len, "history_len", (R,), torch.int32, dev)
            keep += [history, history_len]
            a.history, a.history_stride, a.history_cols = ptr(history), history.stride(0), history.shape[1]
            a.history_len = ptr(history_len)
            if a.history is None or not history.numel():
                a.history = None
        for name, x in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
            if isinstance(x, torch.Tensor):
                x = _side(x, name, (R,), torch.float32, dev)
                keep.append(x)
                setattr(a, name, ptr(x))
            else:
                setattr(a, name + "_all", float(x))
        out = torch.empty(R, A, dtype=torch.float32, device=dev)
        selected = torch.empty(R, dtype=torch.int32, device=dev)
        if R == 0:
            return out, selected
        a.log_probs, a.out_stride, a.selected = ptr(out), A, ptr(selected)
        lib = _lib.load()
        need = lib.dgl_logits_workspace_floats(ctypes.byref(a))
        with _on(dev):
            ws = torch.empty(need, dtype=torch.float32, device=dev) if need > 0 else None
            check(lib.dgl_logits_process(ctypes.byref(a), ptr(ws), _stream(dev)), "dgl_logits_process")
        return out, selected
