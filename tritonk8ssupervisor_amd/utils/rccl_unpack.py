"""An RCCL built from source for this host's GPU alone, used by the fabric check's ranks.

ROCm ships ``librccl.so`` with its device code compressed for every GPU target it supports; the
HIP runtime inflates all of it in every process that first launches an RCCL kernel, which is
~1.7 s of every ``ncclCommInit*`` on the MI355X (docs/benchmarks-history.md). An RCCL that the
operator builds from its public source for gfx950 only, without offload compression, has nothing
to inflate. This module keeps such a build beside the tk8s tree and says whether it is current:

    python3 -m tritonk8ssupervisor_amd.utils.rccl_unpack /path/to/built/librccl.so.1

copies it to ``build/rccl-<arch>/librccl.so.1`` (read-only to pods, like the rest of the install)
and keys it to the installed library (path, size, mtime), so that a ROCm upgrade makes it stale.
The fabric check's ranks load it through ``LD_LIBRARY_PATH`` (``fabric.FabricCheck``) and use the
installed library whenever there is none or it is stale. ``TK8S_RCCL_UNPACKED=0`` turns it off.
The installed library itself is never opened or taken apart.
"""
from __future__ import annotations

import json
import os
import shutil
import struct
from pathlib import Path

from .build_native import ARCH, REPO, ROCM

OUT = REPO / "build" / f"rccl-{ARCH}"
LIB_NAME = "librccl.so.1"


def installed_library() -> Path | None:
    for p in (ROCM / "lib" / LIB_NAME, ROCM / "lib" / "librccl.so"):
        if p.exists():
            return p.resolve()
    return None


def elf_section(path: Path, name: str) -> tuple[int, int] | None:
    """(file offset, size) of section ``name`` of a 64-bit little-endian ELF file; None for a file
    that is not one, or is truncated or malformed."""
    try:
        return _elf_section(path, name)
    except (struct.error, IndexError, ValueError, UnicodeDecodeError):
        return None


def _elf_section(path: Path, name: str) -> tuple[int, int] | None:
    with open(path, "rb") as f:
        eh = f.read(64)
        if eh[:4] != b"\x7fELF" or eh[4] != 2 or eh[5] != 1:
            return None
        shoff, = struct.unpack_from("<Q", eh, 0x28)
        shentsize, shnum, shstrndx = struct.unpack_from("<HHH", eh, 0x3A)
        f.seek(shoff)
        table = f.read(shentsize * shnum)
        sh = [struct.unpack_from("<IIQQQQIIQQ", table, i * shentsize) for i in range(shnum)]
        stroff, strsize = sh[shstrndx][4], sh[shstrndx][5]
        f.seek(stroff)
        names = f.read(strsize)
    for s in sh:
        end = names.index(b"\0", s[0])
        if names[s[0]:end].decode() == name:
            return s[4], s[5]
    return None


def _stamp(src: Path) -> dict:
    st = src.stat()
    return {"source": str(src), "size": st.st_size, "mtime_ns": st.st_mtime_ns, "arch": ARCH}


def library_dir() -> Path | None:
    """The directory of the operator's build when it is current for the installed RCCL, else None."""
    if os.environ.get("TK8S_RCCL_UNPACKED", "1") == "0":
        return None
    src = installed_library()
    try:
        stamp = json.loads((OUT / "stamp.json").read_text())
    except (OSError, ValueError):
        return None
    if src is None or stamp != _stamp(src) or not (OUT / LIB_NAME).is_file():
        return None
    return OUT


def unpack() -> dict:
    """Whether a current build is there; nothing is made (that takes RCCL's source: ``adopt``)."""
    if library_dir() is not None:
        return {"ok": True, "path": str(OUT / LIB_NAME), "changed": False}
    return {"ok": False, "why": "no RCCL built from source for this GPU was given; the installed one is used"}


def adopt(built: Path) -> dict:
    """Keep ``built`` (a librccl the operator compiled from source) as the fabric ranks' library."""
    src = installed_library()
    if src is None:
        return {"ok": False, "why": "no librccl under ROCm"}
    if built.resolve().is_relative_to(ROCM.resolve()):
        return {"ok": False, "why": f"{built} is the installed library, not a build from source"}
    if not built.is_file() or elf_section(built, ".hip_fatbin") is None:
        return {"ok": False, "why": f"{built} is not a library with HIP device code"}
    OUT.mkdir(parents=True, exist_ok=True)
    tmp = OUT / f".{LIB_NAME}.{os.getpid()}"
    shutil.copyfile(built, tmp)
    tmp.chmod(0o755)
    os.replace(tmp, OUT / LIB_NAME)
    (OUT / "stamp.json").write_text(json.dumps(_stamp(src)))
    return {"ok": True, "path": str(OUT / LIB_NAME), "changed": True}


if __name__ == "__main__":
    import sys

    print(json.dumps(adopt(Path(sys.argv[1])) if len(sys.argv) > 1 else unpack()))
