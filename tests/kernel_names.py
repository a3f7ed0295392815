"""Which kernels of the framework a call launches, for tests of sizes that are meant to take one."""
import re

import torch

LIES = ("pieces", "words", "odd")


def kernels(call):
    """The tile kernels of a call in order, each with what its template says of the operands: a name
    and, for tiles, how the operands' rows lie ("ring64 words", "wide pieces", "tile odd", "few")."""
    return [n for n in map(_kind, launches(call)) if n]


def launches(call):
    """The names of all kernels of a call in order, the second time that it is made."""
    from torch.profiler import ProfilerActivity, profile
    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    events = [e for e in p.events() if e.device_type == torch.autograd.DeviceType.CUDA]
    return [e.name for e in sorted(events, key=lambda e: e.time_range.start)]


def _kind(name: str):
    # the names of 16-bit types are not spelled out, and the rest of such a name neither
    if "few_rows_product" in name:
        return "few"
    if "tile_product_shared" in name:
        return "shared"
    tile = re.search(r"tile_product(_wide|_ring)?(?=[<I])", name)
    if not tile:
        return None
    lie = re.search(r"3LieE(\d)|Lie\)(\d)", name)
    lie = LIES[int(lie.group(1) or lie.group(2))]
    if tile.group(1) == "_wide":
        return "wide " + lie
    if tile.group(1) is None:
        return "tile " + lie
    rows = re.search(r"3LieE\dELi(\d)|Lie\)\d, (\d)", name)
    return f"ring{32 * int(rows.group(1) or rows.group(2))} {lie}"
