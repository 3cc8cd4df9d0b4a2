"""Beam search: the best continuations over beams and vocabulary, and a search's state on the device (csrc/beam.cu).

:func:`beam_select` is the selection alone.  A :class:`BeamSearch` keeps what follows from it as well (running scores, next tokens,
parents, finished hypotheses), so that a step needs no look by the host and may be captured in a CUDA graph::

    search = BeamSearch(requests, beams, max_new_tokens, eos=(eos,), device=device)
    while not search.finished():                    # (asks the device; every few steps is enough)
        search.advance(logits)                      # [requests * beams, vocab]
        logits = model(search.tokens, search.parents)
    best = search.result()

A call runs on the current stream of its tensors' device.  A graph reads and writes a search's arrays whenever it is replayed: keep the search as long as the graph.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import c_float, c_int, c_ll, c_void_p

MAX_BEAMS, MAX_KEEP, MAX_EOS = 64, 128, 8
MAX_VOCAB = 1 << 24
_ENTRY: dict = {}
_SCRATCH: dict = {}         # bytes of scratch and launches by requests, beams and tokens


class _State(ctypes.Structure):
    """``State`` of csrc/beam.cu."""
    _fields_ = ([(n, c_void_p) for n in ("scores", "tokens", "parents", "history_token", "history_parent", "pool_score", "pool_step",
                                         "pool_parent", "pool_token", "done", "step")]
                + [("steps", c_int), ("pad", c_int), ("penalty", c_float), ("early", c_int), ("eos_count", c_int), ("eos", c_int * MAX_EOS)])


def _entry():
    if not _ENTRY:
        lib = _lib.load()
        if lib.snu1_beam_state_bytes() != ctypes.sizeof(_State):
            raise _lib.NativeLibraryError(f"{_lib.lib_path()} has searches of another layout: build it again (python -m sensenova_u1_b200.build)")
        P, L, I = c_void_p, c_ll, c_int
        lib.snu1_beam_scratch_bytes.argtypes, lib.snu1_beam_scratch_bytes.restype = (I, I, I), L
        lib.snu1_beam_launches.argtypes = (I, I)
        lib.snu1_beam_step.argtypes = (P, L, I, I, P, I, I, I, P, P, P, P, P, P)
        _ENTRY.update(scratch=lib.snu1_beam_scratch_bytes, launches=lib.snu1_beam_launches, step=lib.snu1_beam_step)
    return _ENTRY


def _check(logits, scores, keep: int, most: int = MAX_KEEP):
    """Requests, beams and tokens of a selection; refuses what the kernels are not made for."""
    if not isinstance(keep, int) or isinstance(keep, bool):
        raise ValueError("keep is a whole number")
    if scores.dim() != 2 or scores.dtype != torch.float32 or not scores.is_contiguous():
        raise ValueError("scores must be contiguous fp32 [requests, beams]")
    requests, beams = scores.shape
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16) or logits.shape[0] != requests * beams:
        raise ValueError(f"logits must be fp32 or bf16 [{requests} x {beams}, vocab], not {tuple(logits.shape)} {logits.dtype}")
    vocab, (row, one) = logits.shape[1], logits.stride()
    if not 1 <= beams <= MAX_BEAMS or not 1 <= keep <= most:
        raise ValueError(f"1 to {MAX_BEAMS} beams, of which 1 to {most} continuations are kept")
    if requests * beams > 65535 or vocab > MAX_VOCAB:
        raise ValueError("too many rows or tokens")
    if keep > beams * vocab:
        raise ValueError(f"{beams} beams of {vocab} tokens have no {keep} continuations")
    if one != 1 and vocab > 1 or (row < vocab and requests * beams > 1):
        raise ValueError("the logits of a row must be contiguous, and rows may not overlap")
    if not logits.is_cuda or scores.device != logits.device:
        raise ValueError("logits and scores must be on one GPU")
    return requests, beams, vocab


def _launch(logits, scores, requests, beams, vocab, keep, out, state) -> None:
    index = logits.get_device()
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return _launch(logits, scores, requests, beams, vocab, keep, out, state)
    entry, size = _entry(), (requests, beams, vocab)
    found = _SCRATCH.get(size)                      # (another thread may empty it at any time)
    if found is None:
        if len(_SCRATCH) > 64:
            _SCRATCH.clear()
        found = _SCRATCH[size] = entry["scratch"](requests * beams, beams, vocab), entry["launches"](beams, vocab)
    count, launches = found
    scratch = torch.empty(count, dtype=torch.uint8, device=logits.device) if count else None
    _lib.LAUNCHES += launches
    rc = entry["step"](logits.data_ptr(), max(logits.stride(0), vocab), logits.dtype == torch.bfloat16, vocab, scores.data_ptr(), requests, beams,
                       keep, None if scratch is None else scratch.data_ptr(), *out, state, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        raise _lib.error("beam_step", rc)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, keep: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``keep`` (default: twice the beams) best continuations of every request by ``scores[r, b] + log_softmax(logits[r * beams + b])[t]``,
    best first: their scores fp32 [requests, keep], beams and tokens int32 [requests, keep].

    ``logits``: fp32 or bf16 [requests * beams, vocab], rows may be slices of wider ones; ``scores``: fp32 [requests, beams].  Scores are compared in
    64 bits, with normalisers that are good to about 1e-7; of equal ones the lower beam comes first, then the lower token (of one beam, the larger logit).  A beam whose score is -inf or not finite, or whose
    logits hold NaN or +inf, has no continuations, and no token of logit -inf is one; places for which none is left hold score -inf, beam
    0, token 0."""
    if keep is None:
        keep = 2 * scores.shape[-1] if scores.dim() == 2 else 0
    requests, beams, vocab = _check(logits, scores, keep)
    out = scores.new_empty((3, requests, keep), dtype=torch.int32)
    if requests:
        at, row = out.data_ptr(), 4 * requests * keep
        _launch(logits, scores, requests, beams, vocab, keep, (at, at + row, at + 2 * row), None)
    best, at, tokens = out.unbind()
    return best.view(torch.float32), at, tokens


class BeamSearch:
    """A batch of searches, ``beams`` each, over at most ``steps`` tokens.

    ``eos``: up to eight tokens that end a hypothesis.  A finished one counts ``score / tokens ** length_penalty``, the ending token among its
    tokens.  ``early_stopping``: False, a request is done when it has ``beams`` finished hypotheses and none of its beams would be better at its
    present length; True, as soon as it has that many; "never", when no beam could be better at any length.  One whose beams have no
    continuation left (logits of NaN, or all -inf) is done too, and they count as they are.

    On the device: ``scores`` fp32 [requests, beams] (-inf: no such beam), ``tokens`` int64 [requests * beams], what the next step reads, and
    ``parents`` int32 [requests * beams], the row of the step before that each row goes on from.  Rows that nobody goes on with keep
    their place.  ``done`` int32 [requests]."""

    def __init__(self, requests: int, beams: int, steps: int, eos=(), length_penalty: float = 1.0, early_stopping=False, device="cuda"):
        if requests < 1 or not 1 <= beams <= MAX_BEAMS or requests * beams > 65535 or steps < 1:
            raise ValueError(f"a search has requests, 1 to {MAX_BEAMS} beams and steps")
        eos = list(dict.fromkeys(int(t) for t in eos))
        if len(eos) > MAX_EOS or any(not 0 <= t < MAX_VOCAB for t in eos):
            raise ValueError(f"up to {MAX_EOS} ending tokens, none negative")
        if early_stopping not in (False, True, "never"):
            raise ValueError('early_stopping is False, True or "never"')
        if not abs(length_penalty) < float("inf"):
            raise ValueError("length_penalty is a number")
        if abs(length_penalty) * math.log2(steps) > 100:
            raise ValueError(f"{steps} tokens ** {length_penalty} leaves fp32: hypotheses could not be compared")
        _entry()
        self.requests, self.beams, self.steps, self.length_penalty = requests, beams, steps, float(length_penalty)
        self.device = torch.device(device)
        make = lambda *shape, dtype=torch.int32, value=0: torch.full(shape, value, dtype=dtype, device=self.device)
        self.scores = make(requests, beams, dtype=torch.float32, value=float("-inf"))
        self.scores[:, 0] = 0
        self.tokens = make(requests * beams, dtype=torch.int64)
        self.parents = torch.arange(requests * beams, dtype=torch.int32, device=self.device)
        self.done = make(requests)
        self._step = make(requests)
        self._history = make(2, steps, requests, beams)                     # tokens, parents
        self._pool_score = make(requests, beams, dtype=torch.float32, value=float("-inf"))
        self._pool = make(3, requests, beams, value=-1)                     # step, parent, token
        early = {False: 0, True: 1, "never": 2}[early_stopping]
        self._state = _State(*(t.data_ptr() for t in (self.scores, self.tokens, self.parents, self._history[0], self._history[1], self._pool_score,
                                                      self._pool[0], self._pool[1], self._pool[2], self.done, self._step)),
                             steps, 0, self.length_penalty, early, len(eos), (c_int * MAX_EOS)(*eos))

    def advance(self, logits: torch.Tensor) -> None:
        """One step, from the logits of the present rows (fp32 or bf16 [requests * beams, vocab]); the first one looks only at every request's first
        row.  A step beyond ``steps`` changes nothing, and ``check_status`` raises after it.  May be captured."""
        # (every beam may end in each of the ending tokens: only among so many are as many that go on as there are beams)
        keep = min(self.beams * max(2, 1 + self._state.eos_count), self.beams * logits.shape[-1])
        requests, beams, vocab = _check(logits, self.scores, keep, MAX_BEAMS * (1 + MAX_EOS))
        _launch(logits, self.scores, requests, beams, vocab, keep, (None, None, None), ctypes.addressof(self._state))

    def finished(self) -> bool:
        """Whether all requests are done or have no step left (waits for the device)."""
        done, step = torch.stack([self.done, self._step]).tolist()
        return all(d or s >= self.steps for d, s in zip(done, step))

    def result(self, best: int = 1) -> list:
        """Per request its ``best`` hypotheses, best first, as (tokens, score); an ending token is the last one.  Beams of requests that are not done
        count as they are.  Waits for the device."""
        if not 1 <= best <= self.beams:
            raise ValueError(f"1 to {self.beams} hypotheses")
        token, parent = self._history.tolist()
        score, pool_score = self.scores.tolist(), self._pool_score.tolist()
        (pool_step, pool_parent, pool_token), done, steps = self._pool.tolist(), self.done.tolist(), self._step.tolist()

        def path(r, step, beam):
            out = []
            for t in range(step, -1, -1):
                out.append(token[t][r][beam])
                beam = parent[t][r][beam]
            return out[::-1]

        out = []
        for r in range(self.requests):
            found = [(pool_score[r][i], path(r, pool_step[r][i] - 1, pool_parent[r][i]) + [pool_token[r][i]])
                     for i in range(self.beams) if pool_step[r][i] >= 0]
            if not done[r] and steps[r]:
                found += [(s / steps[r] ** self.length_penalty, path(r, steps[r] - 1, i)) for i, s in enumerate(score[r]) if s > float("-inf")]
            found.sort(key=lambda f: -f[0])
            out.append([(tokens, s) for s, tokens in found[:best]])
        return out
