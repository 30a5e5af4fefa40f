"""The operator's own RCCL build for the fabric check (utils/rccl_unpack.py).

A build that is given is kept and keyed to the installed library; one that is missing or keyed to
another library is not used (the installed one is). The installed library itself is never opened:
what is read here as a library is this repository's own. On the MI355X the ranks load the build where
one is kept (tests/test_kernels_gpu.py::test_unpacked_rccl_starts_faster_on_a_real_gpu)."""
from __future__ import annotations

import json
from pathlib import Path

import pytest

from tritonk8ssupervisor_amd.utils import rccl_unpack as ru

pytestmark = pytest.mark.skipif(ru.installed_library() is None, reason="no librccl under ROCm")


def test_a_stale_or_disabled_copy_is_not_used(monkeypatch, tmp_path):
    monkeypatch.setattr(ru, "OUT", tmp_path)
    assert ru.library_dir() is None  # none made here
    (tmp_path / ru.LIB_NAME).write_bytes(b"x")
    src = ru.installed_library()
    stamp = ru._stamp(src)
    (tmp_path / "stamp.json").write_text(json.dumps(stamp))
    assert ru.library_dir() == tmp_path
    (tmp_path / "stamp.json").write_text(json.dumps({**stamp, "size": stamp["size"] + 1}))  # RCCL was upgraded
    assert ru.library_dir() is None
    (tmp_path / "stamp.json").write_text(json.dumps(stamp))
    monkeypatch.setenv("TK8S_RCCL_UNPACKED", "0")
    assert ru.library_dir() is None


def test_elf_section_reader(tmp_path, native_build):
    own = Path(native_build["libtk8s"])  # built here from source
    off, size = ru.elf_section(own, ".text")
    assert 0 < off < off + size <= own.stat().st_size
    assert ru.elf_section(own, ".hip_fatbin") is not None and ru.elf_section(own, ".nothing") is None
    (tmp_path / "x").write_bytes(b"not an elf" * 10)
    assert ru.elf_section(tmp_path / "x", ".text") is None


def test_transport_report_of_a_one_rank_log(tmp_path):
    """a 1-rank communicator connects no channel, but its INFO log is there
    -- the report says it was logged, that init completed, and which library the rank loaded."""
    from tritonk8ssupervisor_amd.fabric import rccl_transports

    one = tmp_path / "rank0.log"
    one.write_text("host:1:1 [0] NCCL INFO ROCr version 1.18\nLibrccl path : /x/build/rccl-gfx950/librccl.so.1\n"
                   "host:1:1 [0] NCCL INFO comm 0x1 rank 0 nranks 1 cudaDev 0 busId 5000 - Init COMPLETE\n")
    r = rccl_transports([str(one)])
    assert r["logged"] and r["init_complete"] and r["p2p"] == 0 and r["library"].endswith("rccl-gfx950/librccl.so.1")
    two = tmp_path / "rank1.log"
    two.write_text("host:1:1 [0] NCCL INFO Channel 00/0 : 0[0] -> 1[1] via P2P/IPC\n")
    r = rccl_transports([str(one), str(two), None])
    assert r["p2p"] == 1 and r["logged"]
    assert rccl_transports([str(tmp_path / "none.log")]) == {"p2p": 0, "shm": 0, "net": 0, "collnet": 0,
                                                              "logged": False, "init_complete": False, "library": None}


def test_the_fabric_rank_env_carries_the_unpacked_library_and_huge_page_malloc(monkeypatch, tmp_path):
    """fabric.rccl_rank_env: the unpacked copy asked for (the node's agent prepends ITS copy to the
    rank's LD_LIBRARY_PATH) and glibc's malloc on huge pages (profiles/r5_thp: 318 -> 202 ms
    communicator start), each with its own off-switch; fake GPUs get neither. A GLIBC_TUNABLES
    already set is kept."""
    from tritonk8ssupervisor_amd import fabric
    from tritonk8ssupervisor_amd.utils import rccl_unpack

    monkeypatch.setattr(rccl_unpack, "library_dir", lambda: tmp_path)
    for var in ("TK8S_RCCL_THP", "GLIBC_TUNABLES", "NCCL_DEBUG", "NCCL_DEBUG_SUBSYS", "TK8S_SHORTCUTS", "TK8S_FAULTS",
                "TK8S_GPU_SYNC_TIMEOUT_S", "TK8S_RCCL_BLOCKING", "TK8S_RCCL_PREWARM"):
        monkeypatch.delenv(var, raising=False)
    env, lib = fabric.rccl_rank_env()
    assert lib == tmp_path
    assert {e["name"]: e["value"] for e in env} == {"TK8S_RCCL_UNPACKED": "1",
                                                     "GLIBC_TUNABLES": "glibc.malloc.hugetlb=1"}
    monkeypatch.setenv("GLIBC_TUNABLES", "glibc.malloc.arena_max=2")
    monkeypatch.setenv("NCCL_DEBUG", "INFO")
    env, _ = fabric.rccl_rank_env()
    got = {e["name"]: e["value"] for e in env}
    assert got["GLIBC_TUNABLES"] == "glibc.malloc.arena_max=2:glibc.malloc.hugetlb=1" and got["NCCL_DEBUG"] == "INFO"
    monkeypatch.setenv("TK8S_RCCL_THP", "0")
    assert "GLIBC_TUNABLES" not in {e["name"] for e in fabric.rccl_rank_env()[0]}
    monkeypatch.setenv("TK8S_RCCL_PREWARM", "0")  # the rank's code load on threads: off in the rank too
    assert {"name": "TK8S_RCCL_PREWARM", "value": "0"} in fabric.rccl_rank_env()[0]
    env, lib = fabric.rccl_rank_env(fake=True)
    assert lib is None and [e["name"] for e in env] == ["NCCL_DEBUG"]


def test_the_agent_prepends_its_own_unpacked_copy(tmp_path):
    """the rank's LD_LIBRARY_PATH is the node's copy IN FRONT of the path the node's
    runtime passes on (not replacing it); no request, or no current copy on that node: unchanged."""
    from tritonk8ssupervisor_amd.agent.agent import unpacked_rccl_env

    ask = {"TK8S_RCCL_UNPACKED": "1"}
    assert unpacked_rccl_env(ask, {"LD_LIBRARY_PATH": "/opt/x/lib"}, lambda: tmp_path) == {
        "LD_LIBRARY_PATH": f"{tmp_path}:/opt/x/lib"}
    assert unpacked_rccl_env(ask, {}, lambda: tmp_path) == {"LD_LIBRARY_PATH": str(tmp_path)}
    assert unpacked_rccl_env(ask, {"LD_LIBRARY_PATH": "/opt/x/lib"}, lambda: None) == {}
    assert unpacked_rccl_env({}, {"LD_LIBRARY_PATH": "/opt/x/lib"}, lambda: tmp_path) == {}


def test_the_fabric_rank_env_passes_the_fail_fast_knobs_and_rccl_faults(monkeypatch):
    from tritonk8ssupervisor_amd import fabric

    monkeypatch.setenv("TK8S_FAULTS", "agent.crash@kubenode1, rccl.hang@sweep:1,xgmi.degrade@0-1:0.1,rccl.exit@uid")
    monkeypatch.setenv("TK8S_GPU_SYNC_TIMEOUT_S", "3")
    env, _ = fabric.rccl_rank_env(fake=True)
    got = {e["name"]: e["value"] for e in env}
    assert got["TK8S_FAULTS"] == "rccl.hang@sweep:1,rccl.exit@uid" and got["TK8S_GPU_SYNC_TIMEOUT_S"] == "3"


def test_elf_section_survives_truncated_and_odd_files(tmp_path, native_build):
    """A truncated or malformed library must not raise out of the optional check of a build."""
    own = Path(native_build["libtk8s"]).read_bytes()
    for n in (0, 10, 64, 200, len(own) // 2):
        f = tmp_path / f"t{n}"
        f.write_bytes(own[:n])
        ru.elf_section(f, ".hip_fatbin")  # None or a tuple; never struct.error / IndexError
    odd = bytearray(own[:64]) + bytes(64)
    odd[0x3C:0x3E] = (0xFFFF).to_bytes(2, "little")  # e_shnum far beyond the file
    (tmp_path / "odd").write_bytes(bytes(odd))
    assert ru.elf_section(tmp_path / "odd", ".text") is None


def test_doctor_reports_the_huge_page_mode(tmp_path):
    from tritonk8ssupervisor_amd.doctor import transparent_huge_pages

    f = tmp_path / "enabled"
    f.write_text("always [madvise] never\n")
    assert transparent_huge_pages(str(f))["status"] == "OK" and "madvise" in transparent_huge_pages(str(f))["detail"]
    f.write_text("always madvise [never]\n")
    assert transparent_huge_pages(str(f))["status"] == "WARN"
    assert transparent_huge_pages(str(tmp_path / "missing"))["status"] == "WARN"


def test_an_operators_build_is_kept_and_anything_else_refused(monkeypatch, tmp_path, native_build):
    """A library with device code that was built from source (here: this repository's own) is kept
    and becomes current; the installed RCCL, or a file that is no such library, is refused."""
    monkeypatch.setattr(ru, "OUT", tmp_path / "kept")
    assert not ru.unpack()["ok"]
    assert not ru.adopt(ru.installed_library())["ok"]
    assert not ru.adopt(tmp_path / "missing")["ok"]
    (tmp_path / "text").write_text("no library")
    assert not ru.adopt(tmp_path / "text")["ok"]
    assert ru.library_dir() is None
    assert ru.adopt(Path(native_build["libtk8s"]))["ok"]
    assert ru.library_dir() == tmp_path / "kept" and ru.unpack() == {
        "ok": True, "path": str(tmp_path / "kept" / ru.LIB_NAME), "changed": False}
