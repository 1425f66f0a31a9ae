"""By what a module knows that its weights have changed since it last used them.

``Generator`` and ``Discriminator`` keep images of their weights in the layouts that the kernels read, and make one anew when the
parameter has another address or another version counter.  Torch raises the counter at every write in place, and the optimizers
of this package do so for theirs -- from Python, which the replay of a captured step does not run.  The parameters of a step that
is captured are therefore noted here, and the tag of a noted one never equals an earlier tag: an image of it is made at every use.
That ends with the optimizer, which a graph of its step must not outlive."""
from __future__ import annotations

import weakref

import torch
from torch.utils.weak import WeakTensorKeyDictionary

_noted = WeakTensorKeyDictionary()         # parameter -> the optimizers that have a captured step of it


def note_captured(params, optimizer) -> None:
    """``params`` are written by a step of ``optimizer`` that is being captured into a graph."""
    for p in params:
        owners = _noted.get(p)
        if owners is None:
            owners = _noted[p] = weakref.WeakSet()
        owners.add(optimizer)


def tag(t: torch.Tensor) -> tuple:
    """Equal to an earlier tag of ``t`` if its memory is the same and nothing has written it since."""
    if _noted and _noted.get(t):
        return t.data_ptr(), t._version, object()
    return t.data_ptr(), t._version


def tags(tensors) -> tuple:
    """The tags of ``tensors``."""
    return tuple(map(tag, tensors)) if _noted else tuple((t.data_ptr(), t._version) for t in tensors)


def refuse_capture(what: str, device: int) -> None:
    """For an upload of weights through the host, which no graph would replay."""
    with torch.cuda.device(device):
        capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        raise RuntimeError(f"{what}: the weights have changed, or a captured optimizer step changes them, and their upload goes "
                           "through the host: it cannot be captured into a graph. Call the module once after the last change, before "
                           "the capture; the weights of a captured optimizer step cannot be followed by a captured forward")
