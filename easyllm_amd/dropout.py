"""Where dropout takes its numbers from: a seed and a counter of the calls made so far (base_modules' `get_cuda_rng_tracker` role).

The mask of a call follows from (seed, offset, step) and the elements' indices alone (`include/ezl.h`, ezl_dropout), so nothing random is kept but
these numbers: the backward pass is given the forward's, and a recomputed forward replays them (`recording`, `replaying`; `checkpointing.checkpoint` does, other
recomputations have to, or are refused).  Every call takes the next offset.
Inside a captured graph the offset is frozen; there the kernels add a step that lies in device memory, which whoever replays the graph advances
(`stepping`; `runner.GraphedStep` does), between a replay's end and the next one's start.  Outside one the step is zero, and a graph's first is one, so the two
never draw the same numbers.  A captured graph keeps the numbers it was captured with: it is captured behind `manual_seed` or `set_state`, and a run that
is to go on where it stopped keeps `get_state` and each `GraphedStep.dropout_state`.  Ranks that hold different data are seeded apart by whoever starts them (`manual_seed`).
"""
import contextlib
import threading
from typing import NamedTuple, Optional

import torch


class Draw(NamedTuple):
    """The numbers of one call."""
    seed: int
    offset: int
    step: Optional[torch.Tensor] = None  # int64 [1] on the GPU


class _Thread(threading.local):
    def __init__(self):
        self.records, self.replays, self.steps = [], [], []


_thread = _Thread()
_lock = threading.Lock()
_seed = None
_given = False  # whether it is the caller's; else torch's
_calls = 0
_generation = 0  # how often the draws were started anew or somewhere else


def _follow_torch():
    """Without a seed of dropout's own the draws start anew where torch's seed has changed.  (Lock held.)"""
    global _seed, _calls
    if not _given and _seed != torch.initial_seed():
        _seed, _calls = torch.initial_seed(), 0


def manual_seed(seed):
    """Starts the draws of this process anew.  Until it or `set_state` is called, another seed given to `torch.manual_seed` does (the same one again does
    not: the draws go on)."""
    set_state((seed, 0))


def generation():
    """Another number after every `manual_seed` and `set_state`, which a captured graph does not follow."""
    return _generation


def get_state():
    """(seed, number of calls): what a checkpoint of a training run has to keep, beside the `dropout_state` of each captured step."""
    with _lock:
        _follow_torch()
        return _seed, _calls


def set_state(state):
    global _seed, _given, _calls, _generation
    with _lock:
        _seed, _given, _calls = int(state[0]), True, int(state[1])
        _generation += 1


def next_draw():
    """The numbers of the next call of this thread: new ones, or those of the forward pass that is being recomputed."""
    global _calls
    if _thread.replays:
        try:
            draw = next(_thread.replays[-1])
        except StopIteration:
            raise RuntimeError("a repeated forward makes more dropout calls than the forward whose numbers it takes") from None
    else:
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError("dropout draws new numbers inside a backward pass, where a recomputed forward has to take those of the forward it repeats: "
                               "record the forward's (dropout.recording()) and repeat it under dropout.replaying(), as checkpointing.checkpoint does")
        step = None
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            if not _thread.steps:
                raise RuntimeError("dropout inside a captured graph draws the same mask on every replay unless its step advances: "
                                   "capture with dropout.stepping() (runner.GraphedStep does)")
            step = _thread.steps[-1]
        with _lock:
            _follow_torch()
            draw = Draw((_seed + (_calls >> 32)) & 0xFFFFFFFFFFFFFFFF, _calls & 0xFFFFFFFF, step)
            _calls += 1
    for record in _thread.records:
        record.append(draw)
    return draw


@contextlib.contextmanager
def recording():
    """-> the list of this thread's draws inside the block"""
    draws = []
    _thread.records.append(draws)
    try:
        yield draws
    finally:
        _thread.records.pop()


@contextlib.contextmanager
def replaying(draws):
    """This thread's calls inside the block take `draws`, in order and all of them."""
    draws = list(draws)
    left = iter(draws)
    _thread.replays.append(left)
    try:
        yield
    finally:
        _thread.replays.pop()
    unused = sum(1 for _ in left)
    if unused:  # (a mask of the forward's that the repetition has not applied)
        raise RuntimeError("a repeated forward made %d of %d dropout calls of the forward whose numbers it takes" % (len(draws) - unused, len(draws)))


@contextlib.contextmanager
def stepping(step):
    """Captured calls of this thread inside the block read `step` (int64 [1] on the GPU, 1 or more on every replay)."""
    _thread.steps.append(step)
    try:
        yield
    finally:
        _thread.steps.pop()


def threshold_of(p):
    """An element is dropped where its 16-bit number is below this: p rounded to a multiple of 2^-16."""
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout probability has to be between 0 and 1, but got %r" % (p,))
    return int(p * 65536 + 0.5)
