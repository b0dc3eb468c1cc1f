"""Host-side tile schedule, kept for the ``GroupedMatmul`` contract.

Same semantics as the reference's ``build_tile_schedule``
(src/dispatch/kernels/tile_schedule.py:28-50): per-expert ``block_m``-row tiles
and the exclusive prefix sum ``group_offsets``. The B200 kernels only read
``group_offsets`` (on the device) and derive their own 128-row tiles in-kernel;
the fused layer path never builds this object and never synchronises.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from dispatch_b200 import _lib as L


@dataclass(frozen=True)
class TileSchedule:
    block_m: int
    group_offsets: tuple[int, ...]  # host-side row offsets, len n_experts + 1
    tile_expert: torch.Tensor  # (num_tiles,) int32
    tile_row_start: torch.Tensor  # (num_tiles,) int32
    tile_valid_rows: torch.Tensor  # (num_tiles,) int32, each <= block_m

    @property
    def num_tiles(self) -> int:
        return int(self.tile_expert.shape[0])


def build_tile_schedule(group_sizes: torch.Tensor, block_m: int) -> TileSchedule:
    """Tensors land on group_sizes' device. Reads the sizes on the host, as the
    reference does; prefer the fused path, which keeps offsets on the device."""
    if block_m <= 0:
        raise ValueError(f"block_m must be positive, got {block_m}")
    sizes = [int(s) for s in group_sizes.tolist()]
    offsets = [0]
    te: list[int] = []
    ts: list[int] = []
    tv: list[int] = []
    for expert_id, size in enumerate(sizes):
        for local_start in range(0, size, block_m):
            te.append(expert_id)
            ts.append(offsets[-1] + local_start)
            tv.append(min(block_m, size - local_start))
        offsets.append(offsets[-1] + size)
    dev = group_sizes.device

    def i32(v: list[int]) -> torch.Tensor:
        return torch.tensor(v, dtype=torch.int32, device=dev)

    return TileSchedule(block_m, tuple(offsets), i32(te), i32(ts), i32(tv))


class _Upload:
    """The offsets of a schedule on a device: what was copied, where, and when."""

    __slots__ = ("values", "tensor", "stream", "done")

    def __init__(self, values: tuple[int, ...], device: torch.device):
        self.values = values
        self.tensor = torch.tensor(values, dtype=torch.int32).to(device, non_blocking=True)
        self.stream, self.done = None, None
        if device.type == "cuda":
            self.stream = L.stream_ptr(device)
            self.done = torch.cuda.Event()
            self.done.record(torch.cuda.current_stream(device))

    def __reduce__(self):  # a copied or pickled schedule uploads its own
        return type(None), ()


# read by captured graphs at each replay, whatever becomes of the schedule
_captured_uploads: list[_Upload] = []


def device_offsets(schedule, device: torch.device) -> torch.Tensor:
    """``schedule.group_offsets`` as an int32 device tensor (accepts the
    reference's TileSchedule too: only ``group_offsets`` is read). Uploaded
    once per schedule, device and values; other streams wait for the copy, and
    a captured call's copy is made and finished outside the graph."""
    offsets = schedule.group_offsets
    up = getattr(schedule, "_b200_offsets", None)
    capturing = device.type == "cuda" and torch.cuda.is_current_stream_capturing()
    if up is None or up.tensor.device != device or (up.values is not offsets and up.values != tuple(offsets)):
        values = tuple(offsets)
        up = L.outside_the_capture(device, lambda: _Upload(values, device)) if capturing else _Upload(values, device)
        try:
            object.__setattr__(schedule, "_b200_offsets", up)
        except (AttributeError, TypeError):
            pass
    elif capturing:
        L.outside_the_capture(device, up.done.synchronize)
    elif up.done is not None and up.stream != L.stream_ptr(device):
        here = torch.cuda.current_stream(device)
        here.wait_event(up.done)
        up.tensor.record_stream(here)
    if capturing:
        _captured_uploads.append(up)
    return up.tensor
