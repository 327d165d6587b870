"""Log probabilities of given ids over rows of scores, with rank, entropy and the best
alternatives, and their gradient (rvx_log_probs_*).

Where differentiable_search gives the softmax weights of a few candidates, these take whole rows
of scores — against every row of an index, a batch's other queries, a vocabulary — as a loss and a
ranking: logp is what a contrastive loss sums, rank is the place of the right id.
"""
from __future__ import annotations

from typing import Optional

from . import _lib as L
from .device import Buffer, dtype_code, int32, int64


class LogProbsError(L.RvxError):
    pass


def _check(name, *args):
    try:
        L.call(name, *args)
    except L.RvxError as e:
        raise LogProbsError(e.code, str(e).split(": ", 1)[-1]) from None


def _h(b: Optional[Buffer]):
    return None if b is None else b.handle


def log_probs_device(scores: Buffer, n: int, c: int, temperature: float = 1.0, targets: Optional[Buffer] = None,
                     k: int = 0, logp: Optional[Buffer] = None, rank: Optional[Buffer] = None,
                     entropy: Optional[Buffer] = None, stats: Optional[Buffer] = None,
                     top_ids: Optional[Buffer] = None, top_logp: Optional[Buffer] = None, ld: Optional[int] = None,
                     dtype: str = "f32") -> None:
    """One pass over scores [n][c] of `dtype` (row i at element i * ld, ld = c by default) writes the
    outputs that are given: logp [n] f32 of targets (int64; 0 for a target outside [0, c)), rank [n]
    int64 of the target (-1 without one), entropy [n] f32, stats [n][2] f32 for
    log_probs_backward_device, and the k <= 64 best ids top_ids [n][k] int64 with top_logp [n][k]
    f32 (lowest id first among equals; -1 / -inf past the scores above -inf)."""
    _check("rvx_log_probs_device", scores.handle, dtype_code(dtype), int64(n, "n"), int64(c, "c"),
           int64(c if ld is None else ld, "ld"), temperature,
           _h(targets), int32(k, "k"), _h(logp), _h(rank), _h(entropy), _h(stats), _h(top_ids), _h(top_logp))


def log_probs_backward_device(scores: Buffer, n: int, c: int, temperature: float, stats: Buffer, grad: Buffer,
                              targets: Optional[Buffer] = None, grad_logp: Optional[Buffer] = None,
                              entropy: Optional[Buffer] = None, grad_entropy: Optional[Buffer] = None,
                              ld: Optional[int] = None, ld_grad: Optional[int] = None, dtype: str = "f32") -> None:
    """The gradient by the scores, grad [n][c] of `dtype` (row i at element i * ld_grad), from the
    gradients by logp and by entropy (f32 [n]; None = zeros), with stats and entropy as
    log_probs_device wrote them. grad may be the scores buffer."""
    ld = c if ld is None else ld
    _check("rvx_log_probs_backward_device", scores.handle, dtype_code(dtype), int64(n, "n"), int64(c, "c"), int64(ld, "ld"),
           temperature, _h(targets),
           stats.handle, _h(grad_logp), _h(entropy), _h(grad_entropy), grad.handle,
           int64((ld if grad is scores else c) if ld_grad is None else ld_grad, "ld_grad"))
