"""Beam search over vocabulary-wide logits: a step's selection, the finished
hypotheses, and the models' states that follow the beams.

The reference samples only; this stands beside its decode loops'
(:mod:`graspo_amd.decode_loop`, whose ``generate_beams_with_kv_cache`` runs
the functions here).  A step over ``[groups * beams, V]`` logits is two
launches, nothing waits for the GPU, and all of its state is on the device:

    state = beam_start(groups, beams, device)
    tokens, parents, state, status = beam_step(logits, state, eos_token_id=..., ...)
    reorder_states_(caches, parents, beams, check_status=False)

A beam's best child keeps its slot, so that only the rows of beams that are
replaced are moved.
"""

from __future__ import annotations

import copy
import math
from typing import Any, Callable, NamedTuple

import torch

from . import ops

MAX_BEAMS = 32


class BeamState(NamedTuple):
    """The beams of every group between two steps, on the device."""

    scores: torch.Tensor       # fp32 [G, K], the beams' summed logprobs; -inf: a dead beam
    pool_scores: torch.Tensor  # fp32 [G, K], finished ones' score / length, best first
    pool_rows: torch.Tensor    # int32 [G, K], the row g K + k that ended; -1: empty
    pool_steps: torch.Tensor   # int32 [G, K], at which step; -1: empty
    done: torch.Tensor         # bool [G]
    step: int                  # tokens generated so far


class BeamStep(NamedTuple):
    tokens: torch.Tensor   # int64 [G * K], each slot's next token (pad_token_id where none)
    parents: torch.Tensor  # int32 [G * K], the row that each slot continues
    state: BeamState
    status: torch.Tensor   # int32 [G * K], 0 = ok (ops.STATUS_NAMES)


def _check_beams(what: str, groups: int, beams: int) -> None:
    if groups < 0 or not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"{what}: 1 to {MAX_BEAMS} beams of each group, got {beams} beams and "
                         f"{groups} groups")


def length_of(step: int, length_penalty: float) -> float:
    """What the score of a hypothesis of ``step`` tokens is divided by."""
    try:
        length = float(step) ** float(length_penalty)
    except OverflowError:
        length = math.inf
    if not 0.0 < length < math.inf:
        raise ValueError(f"length_penalty {length_penalty} leaves no finite, positive length at "
                         f"{step} tokens")
    return length


def beam_start(groups: int, beams: int, device, *, all_beams: bool = False) -> BeamState:
    """The state before the first step: one live beam in each group, for the
    prompt's beams are all alike (``all_beams``: they are not)."""
    _check_beams("beam_start", groups, beams)
    scores = torch.full((groups, beams), 0.0 if all_beams else -math.inf, device=device)
    scores[:, 0] = 0.0
    return BeamState(scores, torch.full((groups, beams), -math.inf, device=device),
                     torch.full((groups, beams), -1, dtype=torch.int32, device=device),
                     torch.full((groups, beams), -1, dtype=torch.int32, device=device),
                     torch.zeros((groups,), dtype=torch.bool, device=device), 0)


def beam_step(logits: torch.Tensor, state: BeamState, *, eos_token_id: int, pad_token_id: int,
              length_penalty: float = 1.0, early_stopping: bool = False,
              allow_mask: torch.Tensor | None = None, tokens_out: torch.Tensor | None = None,
              parents_out: torch.Tensor | None = None) -> BeamStep:
    """One step of every group: of the 2 K best ``score + log_softmax(logits)``
    over its K beams and the vocabulary, the finished ones among the first K
    join the pool at score / (tokens so far) ** ``length_penalty``, and the
    first K others become the beams.  A group is done when its pool is full and
    no live beam's score, divided by the present length, is above the pool's
    last (``early_stopping``, a bool: when it is full).  ``logits``: [G * K, V] or
    [G, K, V] (bf16, fp16, fp32; beams may share a row by a stride of 0).
    ``allow_mask``: as :func:`ops.sample`'s, tokens that may follow; the softmax
    is over all."""
    G, K = state.scores.shape
    _check_beams("beam_step", G, K)
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"beam_step: logits must be float32, bfloat16 or float16, got "
                         f"{logits.dtype}")
    if logits.dim() not in (2, 3) or logits.shape[:-1] not in ((G * K,), (G, K)):
        raise ValueError(f"beam_step: expected logits [{G * K}, V] or [{G}, {K}, V], got "
                         f"{tuple(logits.shape)}")
    if logits.shape[-1] > 1 and logits.stride(-1) != 1:
        logits = logits.contiguous()
    new, status = ops.beam_step(
        logits, *state[:5], eos_token_id=eos_token_id, pad_token_id=pad_token_id,
        length=length_of(state.step + 1, length_penalty), step=state.step,
        early_stopping=early_stopping, allow_mask=allow_mask, tokens_out=tokens_out,
        parents_out=parents_out)
    return BeamStep(new.tokens, new.parents, BeamState(*new[2:], state.step + 1), status)


class BeamOutput(NamedTuple):
    scores: torch.Tensor   # fp32 [G, n], score / length ** length_penalty, best first
    lengths: torch.Tensor  # int32 [G, n], tokens, the end-of-sequence one among them
    tokens: torch.Tensor   # int64 [G, n, T], padded behind


def beam_finish(state: BeamState, tokens: torch.Tensor, parents: torch.Tensor, *,
                eos_token_id: int, pad_token_id: int, length_penalty: float = 1.0,
                num_return: int = 1) -> BeamOutput:
    """The ``num_return`` best hypotheses of each group: the pool's, and those
    of the beams that still go on.  ``tokens`` (int64) and ``parents`` (int32)
    are the steps', [state.step, G * K]."""
    G, K = state.scores.shape
    _check_beams("beam_finish", G, K)
    if not 1 <= num_return <= K:
        raise ValueError(f"beam_finish: num_return must be 1 to {K}, got {num_return}")
    if tuple(tokens.shape) != (state.step, G * K) or tokens.shape != parents.shape:
        raise ValueError(f"beam_finish: expected tokens and parents [{state.step}, {G * K}], got "
                         f"{tuple(tokens.shape)} and {tuple(parents.shape)}")
    return BeamOutput(*ops.beam_finish(
        *state[:5], tokens, parents, length=length_of(max(state.step, 1), length_penalty),
        eos_token_id=eos_token_id, pad_token_id=pad_token_id, give=num_return))


# ------------------------------------------------------------- models' states

def reorder_states_(states, parents: torch.Tensor, num_beams: int, *,
                    check_status: bool = True) -> None:
    """``t[:] = t[parents]`` of every tensor of ``states``, in place and
    without a second buffer: tensors of any type and strides whose first
    dimension counts the ``G * num_beams`` rows (a view of a cache's filled part
    is one).  ``parents`` (int32 or int64 [G * num_beams]) maps each group's rows
    onto rows of the same group; one that does not raises ``RuntimeError``, for
    which the call waits for the GPU (its row stays as it was).  With
    ``check_status=False`` (a step's own parents), and in a graph capture, it
    does not wait.  States that overlap in memory are refused."""
    if parents.dtype not in (torch.int32, torch.int64) or parents.dim() != 1:
        raise ValueError(f"reorder_states_: parents must be int32 or int64 [rows], got "
                         f"{parents.dtype} {tuple(parents.shape)}")
    if num_beams < 1 or parents.shape[0] % num_beams:
        raise ValueError(f"reorder_states_: {parents.shape[0]} rows are no groups of {num_beams}")
    states = list(states)
    if parents.dtype == torch.int64:
        parents = parents.clamp(-1, parents.shape[0]).to(torch.int32)
    ops.reorder_states_(states, parents.contiguous(), num_beams, check=bool(check_status))


def expand_states(states, num_beams: int) -> list[torch.Tensor]:
    """``t.repeat_interleave(num_beams, dim=0)`` of every tensor: a prompt's
    state for each of its beams."""
    if num_beams < 1:
        raise ValueError(f"expand_states: num_beams must be at least 1, got {num_beams}")
    return ops.expand_states(list(states), num_beams)


def map_states(cache: Any, change: Callable[[list[torch.Tensor]], list[torch.Tensor]]) -> Any:
    """``cache`` (tensors in nested tuples, lists and dicts; None and plain
    values stay) with its tensors replaced by ``change`` of their list."""
    found: list[torch.Tensor] = []

    def collect(c):
        if isinstance(c, torch.Tensor):
            found.append(c)
        elif isinstance(c, dict):
            for v in c.values():
                collect(v)
        elif isinstance(c, (list, tuple)):
            for v in c:
                collect(v)
        elif not (c is None or isinstance(c, (bool, int, float, str))):
            raise TypeError(f"a cache of tensors in tuples, lists and dicts is expected, got "
                            f"{type(c).__name__}")

    collect(cache)
    new = iter(change(found))

    def rebuild(c):
        if isinstance(c, torch.Tensor):
            return next(new)
        if isinstance(c, dict):
            d = copy.copy(c)  # (of its own kind, with what that keeps beside the items)
            for k, v in c.items():
                d[k] = rebuild(v)
            return d
        if isinstance(c, tuple) and hasattr(c, "_fields"):
            return type(c)(*(rebuild(v) for v in c))
        if isinstance(c, (list, tuple)):
            return type(c)(rebuild(v) for v in c)
        return c

    return rebuild(cache)
