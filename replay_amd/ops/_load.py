"""Loader for the in-tree HIP extension (gfx950).

The extension is built in-tree by ``__graft_entry__.build()`` (so the .so
travels to the GPU box with the repo snapshot) via torch.utils.cpp_extension
with PYTORCH_ROCM_ARCH=gfx950.
"""

from __future__ import annotations

import importlib.util
import os
import re
import struct
from pathlib import Path
from typing import Dict

_HERE = Path(__file__).parent
EXT_NAME = "replay_amd_hip"


def _so_path() -> Path:
    return _HERE / f"{EXT_NAME}.so"


def load_extension():
    so = _so_path()
    if not so.exists():
        raise FileNotFoundError(so)
    import torch  # noqa: F401  (registers torch symbols the .so needs)

    spec = importlib.util.spec_from_file_location(EXT_NAME, so)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


#: kernels that must not use scratch memory: a build of the linear-attention pass
#: that spilled registers gave wrong first chunks now and then, by a cause that
#: was not found, and none without spills did
_WITHOUT_SCRATCH = re.compile(r"\d(la_\w+|gemm_tile|join_parts|slope_product)")


def scratch_bytes(library) -> Dict[str, int]:
    """Bytes of scratch memory a lane, for each GPU kernel of a library built
    here (its spilled vector registers and local arrays): what the kernel
    descriptors (symbols ``<kernel>.kd``) of its code objects say."""
    data = Path(library).read_bytes()
    found, magic, at = {}, b"__CLANG_OFFLOAD_BUNDLE__", 0
    while (at := data.find(magic, at)) >= 0:
        (entries,) = struct.unpack_from("<Q", data, at + 24)
        entry = at + 32
        for _ in range(entries):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            target = data[entry + 24 : entry + 24 + length]
            entry += 24 + length
            if b"gfx" in target and size:
                found.update(_descriptors(data[at + offset : at + offset + size]))
        at += len(magic)
    return found


def _descriptors(elf: bytes) -> Dict[str, int]:
    (table,) = struct.unpack_from("<Q", elf, 40)
    width, count = struct.unpack_from("<HH", elf, 58)
    sections = [struct.unpack_from("<IIQQQQIIQQ", elf, table + i * width) for i in range(count)]
    found = {}
    for _, kind, _, _, start, size, link, _, _, each in sections:
        if kind != 11:  # the dynamic symbols
            continue
        names = sections[link][4]
        for symbol in range(start, start + size, each):
            name, _, _, home, value = struct.unpack_from("<IBBHQ", elf, symbol)
            text = elf[names + name : elf.index(b"\0", names + name)].decode()
            if text.endswith(".kd") and 0 < home < count:
                _, _, _, address, offset, *_ = sections[home]
                (private,) = struct.unpack_from("<I", elf, offset + value - address + 4)
                found[text[: -len(".kd")]] = private
    return found


def check_scratch(library) -> None:
    """Raise if a kernel that must not use scratch memory does."""
    used = scratch_bytes(library)
    kept = [name for name in used if _WITHOUT_SCRATCH.search(name)]
    if not kept:
        raise RuntimeError(f"found no kernels to check for register spills in {library}")
    spilled = {name: used[name] for name in kept if used[name]}
    if spilled:
        raise RuntimeError(f"kernels that must not spill registers use scratch memory (bytes a lane): {spilled}")


def build_extension(verbose: bool = True):
    """Compile the HIP sources for gfx950 into replay_amd/ops/replay_amd_hip.so."""
    os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")
    from torch.utils.cpp_extension import load

    src_dir = _HERE / "hip"
    # exclude torch-hipify's generated *_hip.hip copies of our sources
    sources = sorted(
        str(p) for p in src_dir.glob("*.hip") if not p.name.endswith("_hip.hip")
    ) + sorted(str(p) for p in src_dir.glob("*.cpp"))
    if not sources:
        raise RuntimeError(f"No HIP sources under {src_dir}")
    build_dir = _HERE / "build"
    build_dir.mkdir(exist_ok=True)
    module = load(
        name=EXT_NAME,
        sources=sources,
        extra_cflags=["-O3"],
        # no packed fp32 arithmetic: hipcc forms it from ordinary float code, and
        # some of its forms have given wrong results on this hardware
        extra_cuda_cflags=[
            "-O3", "--offload-arch=gfx950", "-std=c++17",
            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        ],
        build_directory=str(build_dir),
        verbose=verbose,
    )
    # copy the built .so in-tree so it snapshots to the GPU box
    built = build_dir / f"{EXT_NAME}.so"
    if built.exists():
        import shutil

        check_scratch(built)
        shutil.copy2(built, _so_path())
    return module
