"""The layer probe's way into the validation payload: commands and options (no GPU here)."""
import os

import pytest

from tritonk8ssupervisor_amd import earlyburn
from tritonk8ssupervisor_amd.cli import main as cli


def test_the_payload_asks_for_the_layer_only_when_told(monkeypatch):
    monkeypatch.delenv("TK8S_FAKE_GPUS", raising=False)
    assert "--layer" not in earlyburn.default_validation_command()
    for peers in (False, True):
        cmd = earlyburn.default_validation_command(peers=peers, layer=True)
        assert os.path.basename(cmd[0]) == "tk8s-probe" and cmd[-1] == "--layer" and ("--peers" in cmd) == peers


@pytest.mark.parametrize("gpus", [[0], [0, 1], list(range(8))])
def test_the_host_burnin_keeps_the_tool_that_knows_the_layer(monkeypatch, gpus):
    monkeypatch.delenv("TK8S_FAKE_GPUS", raising=False)
    cmd = earlyburn.host_burnin_command(earlyburn.default_validation_command(peers=False, layer=True), gpus)
    assert os.path.basename(cmd[0]) == "tk8s-probe" and "--layer" in cmd and ("--peers" in cmd) == (len(gpus) > 1)


def test_the_pulls_alone_run_no_layer(monkeypatch):
    monkeypatch.delenv("TK8S_FAKE_GPUS", raising=False)
    cmd = earlyburn.host_burnin_command(earlyburn.default_validation_command(peers=False, layer=True), [0, 1])
    assert "--layer" not in earlyburn.hip_peer_command(cmd)


def test_setup_takes_the_option(tmp_path):
    argv = ["setup", "--answers", "a.json", "--layer"]
    assert cli._fast_setup_args(argv).layer is True
    assert cli._fast_setup_args(argv[:-1]).layer is False


def test_the_early_burnin_leaves_such_a_setup_to_the_orchestrator(tmp_path):
    (tmp_path / "a.json").write_text('{"nodes": 1, "package": "mi355x-1gpu"}')
    env = {"TK8S_FAKE_GPUS": "1"}
    assert earlyburn.plan(["--answers", "a.json"], env, str(tmp_path)) is not None
    assert earlyburn.plan(["--answers", "a.json", "--layer"], env, str(tmp_path)) is None


def test_setup_passes_it_on(tmp_path, monkeypatch):
    from tritonk8ssupervisor_amd import orchestrator

    monkeypatch.delenv("TK8S_FAKE_GPUS", raising=False)
    s = orchestrator.Setup(orchestrator.Workspace(tmp_path), layer=True)
    assert "--layer" in s._validation_command()
    assert "--layer" not in orchestrator.Setup(orchestrator.Workspace(tmp_path))._validation_command()
