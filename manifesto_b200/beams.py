"""Beam search's selection over beams and vocabulary, on device addresses.

One step of beam search: ``BeamSelect.run`` chooses the continuations, ``paged.PageBook.fork``
reorders the page tables by the chosen parents and ``paged.PageCopy.run`` copies the pages
that rows no longer share; then the step goes on as ``manifesto_b200.paged`` describes, with
``paged.PrefixAttention`` for the beams of a prompt.  ``include/mfcuda.h`` has the formulas (K11).
"""
from __future__ import annotations

import ctypes

from . import _abi
from .backend import stream_handle
from .dtype import DType
from .paged import _Handle, _raise


class BeamSelect(_Handle):
    """The n_out best continuations of each batch entry (mf_beam_select_*).

    Holds the workspace for batches of up to ``max_batch``, so one object serves one stream
    at a time.  ``row_stride`` is the elements from one row of logits to the next."""

    _destroy = "mf_beam_select_destroy"

    def __init__(self, dtype: DType, vocab: int, beams: int, n_out: int, max_batch: int, row_stride: int | None = None,
                 end_token: int = -1):
        self.config = _abi.BeamSelectConfig(int(dtype), int(vocab), int(beams), int(n_out), int(max_batch), int(end_token),
                                            int(vocab if row_stride is None else row_stride))
        self._create("mf_beam_select_create", ctypes.byref(self.config))
        self._select = _abi.lib().mf_beam_select_run

    def run(self, logits: int, scores: int, batch: int, scores_after: int, tokens: int, parents: int, ended: int = 0,
            ended_after: int = 0, stream=None) -> None:
        """scores, tokens, parents (rows of this call) and ended flags of the chosen, [batch, n_out] each."""
        rc = self._select(self._open(), logits, scores, ended, batch, scores_after, tokens, parents, ended_after,
                          stream if stream is None else stream_handle(stream))
        if rc:
            _raise("mf_beam_select_run", rc)
