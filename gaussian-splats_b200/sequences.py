"""Packed batches of sequences, as the sequence operators take them.

A refiner sees a scene's Gaussians as a sequence of tokens. A batch of scenes of
different sizes is packed: the sequences' tokens follow one another along the
first axis of every tensor, and a :class:`PackedSequences` says where each one
begins. It is built once a batch and handed to every operator of the step.
"""

from __future__ import annotations

import ctypes
from collections.abc import Sequence

import torch

from . import native

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # GS_FLOAT32, ...


class PackedSequences:
    """The layout of a packed batch: ``lengths[b]`` tokens of sequence ``b``
    after those of the sequences before it. Lengths are host integers, zero
    allowed. ``offsets`` (int64, one more than sequences) and the tables that
    the kernels read live on ``device``; they are copied there once, here."""

    def __init__(self, lengths: Sequence[int], device="cuda"):
        self.lengths = tuple(int(n) for n in lengths)
        if not self.lengths:
            raise ValueError("PackedSequences needs at least one sequence")
        if min(self.lengths) < 0:
            raise ValueError(f"sequence lengths must be >= 0, got {min(self.lengths)}")
        self.total = sum(self.lengths)
        check_tokens(self.total, "PackedSequences")
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        length = torch.tensor(self.lengths, dtype=torch.int64)
        offsets = torch.zeros(len(self.lengths) + 1, dtype=torch.int64)
        torch.cumsum(length, 0, out=offsets[1:])
        tile = native.SEQUENCE_TILE
        tiles = (length + tile - 1) // tile
        starts = torch.zeros(len(self.lengths) + 1, dtype=torch.int64)
        torch.cumsum(tiles, 0, out=starts[1:])
        sequence = torch.repeat_interleave(torch.arange(len(self.lengths)), tiles)
        begin, end = offsets[sequence], offsets[sequence + 1]
        within = torch.arange(len(sequence)) - starts[sequence]
        table = torch.stack((begin, end, begin + tile * within, sequence), 1)
        self.offsets = offsets.to(self.device)
        self.tiles = table.to(torch.int32).to(self.device)
        self.tile_starts = starts.to(torch.int32).to(self.device)
        self.num_tiles = len(sequence)
        self._stream = _raw_stream(self.device)

    def __len__(self) -> int:
        return len(self.lengths)


def _raw_stream(device: torch.device) -> int | None:
    return torch._C._cuda_getCurrentRawStream(device.index) if device.type == "cuda" else None


def check_tokens(tokens: int, what: str) -> None:
    """Refuses more tokens than the kernels' 32-bit positions count."""
    if tokens > native.MAX_SEQUENCE_TOKENS:
        raise ValueError(f"{what}: {tokens} tokens, at most {native.MAX_SEQUENCE_TOKENS} are "
                         "supported")


def check_packed(packed: PackedSequences | None, tokens: int, device: torch.device,
                 what: str) -> None:
    """Refuses a layout that does not describe ``tokens`` rows on ``device``."""
    if packed is None:
        return
    if packed.total != tokens:
        raise ValueError(f"{what}: the packed sequences hold {packed.total} tokens, the tensors "
                         f"{tokens}")
    if packed.device != device:
        raise RuntimeError(f"{what}: packed sequences on {packed.device}, tensors on {device}")


def tile_arguments(packed: PackedSequences | None, tokens: int) -> dict:
    """The layout's fields of an operator's arguments: without one, the rows
    are one sequence and its tiles follow from their number."""
    if packed is None:
        return {"sequences": 1, "num_tiles": -(-tokens // native.SEQUENCE_TILE)}
    if packed._stream != _raw_stream(packed.device):
        # A caller cannot know of these tables: their memory is kept until this
        # stream's work is done, also if the layout is dropped before.
        for table in (packed.tiles, packed.tile_starts):
            table.record_stream(torch.cuda.current_stream(packed.device))
    return {"sequences": len(packed), "num_tiles": packed.num_tiles,
            "tiles": packed.tiles.data_ptr() if packed.num_tiles else None,
            "tile_starts": packed.tile_starts.data_ptr()}


def element_type(dtype: torch.dtype, what: str, allowed=(torch.float32, torch.bfloat16,
                                                         torch.float16)) -> int:
    """The library's code of an element type."""
    if dtype not in allowed:
        names = ", ".join(str(d).removeprefix("torch.") for d in allowed)
        raise ValueError(f"{what}: {dtype} is not supported (only {names})")
    return _DTYPES[dtype]


def call(name: str, device: torch.device, *arguments) -> None:
    """Calls a library function on the device's current stream; raises for a
    status other than success."""
    stream = ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(device.index))
    function = getattr(native.lib(), name)
    if device.index == torch._C._cuda_getDevice():
        status = function(*arguments, stream)
    else:
        with torch.cuda.device(device):
            status = function(*arguments, stream)
    if status:
        native.check(status, name)


def changed_in_place(*tensors: torch.Tensor | None) -> None:
    """Tells autograd that a library call wrote to tensors of its caller: a graph
    that saved one before then refuses its backward instead of using what is there now."""
    torch.autograd.graph.increment_version(tuple(t for t in tensors if t is not None))


def address(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def check_cuda(what: str, **tensors: torch.Tensor | None) -> torch.device:
    """The CUDA device of the tensors; raises unless all are on the same one."""
    present = [t for t in tensors.values() if t is not None]
    index = present[0].get_device()
    if index >= 0 and all(t.get_device() == index for t in present):
        return present[0].device
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{what} runs on CUDA devices only (there is no CPU path); {name} "
                               f"is on {t.device}")
        if device is None:
            device = t.device
        elif t.device != device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, the others on {device}")
    return device
