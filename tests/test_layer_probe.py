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


# ---- its checks on the host, and mistakes planted in what they are given ------------------------------


@pytest.fixture(scope="module")
def nat(native_build):
    from tritonk8ssupervisor_amd.ops import native

    return native()


def _bf16(x):
    import numpy as np

    u = np.asarray(x, dtype=np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)  # to nearest, ties to even


def _value(u):
    import numpy as np

    return (u.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


@pytest.mark.parametrize("n", [128, 128 * 128])
@pytest.mark.parametrize("spread", [1.0, 1e-30, 1e36, 0.0])
def test_rounded_values_are_held_to_every_byte(nat, n, spread):
    import numpy as np

    from tritonk8ssupervisor_amd.ops import reference as ref

    rng = np.random.default_rng(n)
    source = _bf16(rng.normal(size=n) * spread)
    source[:64] = _bf16(np.arange(-32, 32) / 32 * spread)  # ties among them
    values, scales = ref.fp8_quantize(_value(source).reshape(n // 128, 128), block_rows=n // 128)
    values, scale = values.ravel(), int(scales[0, 0])
    assert nat.layer_rounding_error(source, values, scale) == 0
    for wrong in (scale - 1, scale + 1):
        assert nat.layer_rounding_error(source, values, wrong) > 1
    for at, mask in ((0, 1), (n // 2, 1), (n - 1, 8), (n - 1, 0x7F)):
        planted = values.copy()
        planted[at] ^= mask
        assert nat.layer_rounding_error(source, planted, scale) > 1, (at, mask)
    other = values.copy()
    other[[1, 40]] = other[[40, 1]]
    assert spread == 0 or nat.layer_rounding_error(source, other, scale) > 1
    with pytest.raises(ValueError):
        nat.layer_rounding_error(source, values[:-1], scale)


@pytest.mark.parametrize("rows", [128, 4096])
def test_the_norms_weight_gradient_is_held_to_its_sum(nat, rows):
    import numpy as np

    rng = np.random.default_rng(rows)
    dy, h = _bf16(rng.normal(size=rows)), _bf16(rng.normal(size=rows) * 3)
    rstd = rng.uniform(0.2, 1, rows).astype(np.float32)
    terms = _value(dy) * _value(h) * rstd
    want, allowed = terms.sum(), (rows + 4) * 2.0 ** -24 * np.abs(terms).sum()
    assert nat.layer_weight_sum_error(np.float32(want), dy, h, rstd) <= 1
    for planted in (want + 2 * allowed, want - 2 * allowed, want + np.abs(terms).sum() / 100, float("nan")):
        assert nat.layer_weight_sum_error(np.float32(planted), dy, h, rstd) > 1, planted
    with pytest.raises(ValueError):
        nat.layer_weight_sum_error(0.0, dy, h, rstd[:-1])


def test_a_machines_share_of_the_host_burnin_is_judged_by_its_layer_too():
    """A GPU whose matrix cores failed does not pass for a bad link from another machine's GPU."""
    from tritonk8ssupervisor_amd.burnin import split_host_result

    def device(i, layer_ok, digest_ok=True, link_ok=True):
        fine = {"ok": True}
        return {"device": i, "ok": layer_ok and digest_ok, "hbm": fine, "md5": fine, "digest_ok": True, "copy": fine,
                "layer": {"ok": layer_ok, "digest": "d"}, "layer_digest_ok": digest_ok,
                "peers": [{"ok": link_ok, "src_device": 1 - i, "dst_device": i}]}

    def share(**kw):
        return split_host_result({"ok": True, "layer_expected": "d", "devices": [device(0, **kw), device(1, True)]}, [4, 5], [4], {"pulls": []})

    for link_ok in (True, False):
        good = share(layer_ok=True, link_ok=link_ok)
        assert good["layer"]["digest"] == good["layer_expected"] == "d"
        assert not share(layer_ok=False, link_ok=link_ok)["ok"]
        assert not share(layer_ok=True, digest_ok=False, link_ok=link_ok)["ok"]
    assert share(layer_ok=True, digest_ok="unpinned")["ok"]
