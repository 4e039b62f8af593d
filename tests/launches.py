"""Which kernels an entry of the layers launches, without a GPU: the entries'
objects linked against csrc/hip_names.c, which notes each launch."""
from __future__ import annotations

import ctypes
import re
import subprocess
from contextlib import contextmanager
from typing import NamedTuple

from turbinator_c_amd import build, layers, native

SOURCES = ("expert_rows", "embed", "int8", "mx4")
TYPES = {"f": "f32", "DF16b": "bf16", "DF16_": "f16"}
ENTRIES = ("expert_rows", "expert_sum", "embed", "int8", "mx4")


class Launch(NamedTuple):
    name: str  # as kernel_of gives it
    grid: tuple
    block: tuple


class Dim3(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint) for n in "xyz"]


def load(folder):
    lib, stub = folder / "names.so", folder / "names.o"
    objects = [build.BUILD / f"{name}.hip.o" for name in SOURCES]
    subprocess.run(["gcc", "-O1", "-fPIC", "-c", str(build.GPU_CHECKS / "hip_names.c"), "-o",
                    str(stub)], check=True)
    subprocess.run(["g++", "-shared", "-o", str(lib), *map(str, objects), str(stub)], check=True)
    return native._load(lib, {n: v for n, v in native.HIP_SIGNATURES.items()
                              if n.startswith(tuple(f"tb_hip_{x}" for x in ENTRIES))})


def kernel_of(mangled: str) -> str:
    """A kernel's name and template arguments: "tile_kernel bf16 0 2 4 6 4 2"."""
    found = re.fullmatch(r"_ZN12_GLOBAL__N_1(\d+)(.*)", mangled)
    size = int(found[1])
    name, rest = found[2][:size], found[2][size:]
    words = [name]
    if rest.startswith("I"):
        typed = re.match(r"I(f|DF16b|DF16_)?((?:L[a-zA-Z_0-9]+?E)*)", rest)
        words += [TYPES[typed[1]]] if typed[1] else []
        words += re.findall(r"(\d+)E", re.sub(r"L(?:NS_\d+\w+?E|[a-z])(?=\d+E)", "", typed[2]))
    return " ".join(words)


@contextmanager
def noted(lib):
    """layers' entries go to `lib`; yields a function that runs one of them and
    returns its launches."""
    own, layers.hip_lib = layers.hip_lib, lambda: lib

    def run(entry, **args):
        count = ctypes.c_int.in_dll(lib, "names_launches")
        count.value = 0
        assert getattr(layers, entry)(**args) == 1
        n = count.value
        assert 0 < n <= 64
        names = [kernel_of(v.decode()) for v in (ctypes.c_char_p * 64).in_dll(lib, "names_of")[:n]]
        sizes = [[(d.x, d.y, d.z) for d in (Dim3 * 64).in_dll(lib, at)[:n]]
                 for at in ("names_grids", "names_blocks")]
        return [Launch(*v) for v in zip(names, *sizes)]

    try:
        yield run
    finally:
        layers.hip_lib = own
