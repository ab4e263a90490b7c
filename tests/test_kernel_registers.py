"""Registers of the built kernels: the persistent engine's two kernels never end,
so every kernel has to find room beside them whatever the order. The counts stand
in the metadata of the code objects inside the built library."""
import re
import struct
from pathlib import Path

import msgpack
import pytest

import accl_amd._core as core

CSRC = Path(core.__file__).parent / "csrc" / "gpu"
REGISTERS = 512  # of a SIMD, which its waves share, in steps of 8
CUS, SIMDS, ENGINES = 256, 4, 32  # SIMDs of a compute unit, shader engines


def _code_objects(data):
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    at = data.find(magic)
    while at >= 0:
        n, = struct.unpack_from("<Q", data, at + 24)
        p = at + 32
        for _ in range(n):
            offset, size, name = struct.unpack_from("<QQQ", data, p)
            triple = data[p + 24:p + 24 + name]
            p += 24 + name
            if size and b"gfx950" in triple:
                yield data[at + offset:at + offset + size]
        at = data.find(magic, at + 24)


def _kernels(elf):
    table, = struct.unpack_from("<Q", elf, 40)
    size, n = struct.unpack_from("<HH", elf, 58)
    for i in range(n):
        kind, = struct.unpack_from("<I", elf, table + i * size + 4)
        if kind != 7:  # notes
            continue
        p, length = struct.unpack_from("<QQ", elf, table + i * size + 24)
        end = p + length
        while p < end:
            name, desc, _ = struct.unpack_from("<III", elf, p)
            at = p + 12 + (name + 3) // 4 * 4
            if elf[p + 12:p + 18] == b"AMDGPU":
                yield from msgpack.unpackb(elf[at:at + desc])["amdhsa.kernels"]
            p = at + (desc + 3) // 4 * 4


def _kernel(part):
    with open(core.__file__, "rb") as f:
        data = f.read()
    found = [k for elf in _code_objects(data) for k in _kernels(elf)
             if part in k[".name"]]
    assert len(found) == 1, [k[".name"] for k in found]
    # .vgpr_count has both kinds of vector registers
    return (found[0][".max_flat_workgroup_size"],
            (found[0][".vgpr_count"] + 7) // 8 * 8)


def _number(header, pattern):
    return int(re.search(pattern, (CSRC / header).read_text()).group(1))


def _groups(wgs):
    """Mover workgroups of an engine that is sized `wgs`."""
    most = _number("engine.hpp", r"MOVER_GROUPS_MAX = (\d+);")
    return max(1, min(most, -(-wgs // 4)))


def test_two_workgroups_share_a_compute_unit():
    """Any two: two schedulers, a scheduler and a mover group, two groups."""
    threads, mover = _kernel("accl_mover_kernel")
    assert threads == _number("engine.hpp", r"MOVER_THREADS = (\d+);")
    waves = threads // 64 // SIMDS  # on each SIMD
    assert waves * mover <= REGISTERS // 2
    assert _kernel("accl_scheduler_kernel")[1] <= REGISTERS // 2


@pytest.mark.parametrize("ranks", [0, 1, 2, 4])
def test_engines_find_room_beside_each_other(ranks):
    """An engine of the default size, those of the ranks of a test beside it (of
    128 in all), and a scheduler each, which may all be dealt to one shader
    engine: resident together whatever the order."""
    places = 2 * CUS // ENGINES
    fleet = _groups(_number("gpudevice.hpp", r"engine_wgs_ = (\d+);"))
    of_rank = _groups(max(16, 128 // ranks)) if ranks else 0
    # a fleet is dealt out evenly to 8 dies and there to 4 shader engines
    most = [-(-(-(-g // 8)) // 4) for g in [fleet] + [of_rank] * ranks]
    assert sum(most) + 1 + ranks <= places


def test_the_largest_fleet_leaves_room():
    assert -(-_groups(10 ** 6) // ENGINES) + 1 <= 2 * CUS // ENGINES
