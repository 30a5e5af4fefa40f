"""The layer probe on the GPU: its own checks of the 8-bit layer, alone and through tk8s-probe."""
import json
import subprocess

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tritonk8ssupervisor_amd.ops import native

    return native()


@pytest.mark.parametrize("rows,width", [(128, 128), (256, 640), (1152, 1024), (2048, 2432), (4096, 4096)])
def test_a_step_of_the_layer_holds_its_bounds(nat, rows, width):
    r = json.loads(nat.layer_probe(rows, width, 7, 2, 0))
    assert r["ok"], r
    assert r["error"] <= 1 and r["steps_that_differ"] == 0 and set(r["errors"]) == {
        "norm", "rounding", "forward", "input_gradient", "weight_gradient", "norm_gradient"}
    # each compared something: results are rounded but for the 32-bit ones, whose sums can be exact
    assert all(e > 0 or name == "weight_gradient" for name, e in r["errors"].items()), r["errors"]
    again = json.loads(nat.layer_probe(rows, width, 7, 1, 0))
    assert again["digest"] == r["digest"]
    assert json.loads(nat.layer_probe(rows, width, 8, 1, 0))["digest"] != r["digest"]


def test_it_is_a_step_of_the_operators(nat):
    """The probe's step, made again from its inputs through the Python entry points: the same digest."""
    from tritonk8ssupervisor_amd.ops import fp8, reference as ref

    def fill(rows, cols, seed):
        x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
        nat.layer_fill(x.data_ptr(), x.numel(), seed, torch.cuda.current_stream().cuda_stream)
        return x

    rows, width, seed = 256, 512, 11
    x, res, weight, w, g = fill(rows, width, seed), fill(rows, width, seed + 1), fill(1, width, seed + 2)[0], fill(width, width, seed + 3), fill(rows, width, seed + 4)
    assert torch.equal(x, (x.float() * 32).round().div(32).bfloat16()) and x.min() == -4 and x.max() == 127 / 32
    assert abs(x.float().mean().item()) < 0.1 and not torch.equal(x, res)
    n = fp8.rms_norm(x, weight, residual=res, eps=1e-5, normed=True)
    y = fp8.matmul(n.quantized, fp8.quantize(w, layout="tiles"))
    g_rows, g_cols = fp8.quantize(g, layout="both")
    dn = fp8.matmul(g_rows, fp8.quantize(w, layout="columns"))
    dw = fp8.matmul(g_cols, fp8.quantize(n.y, layout="columns"), dtype=torch.float32)
    dx, dweight = fp8.rms_norm_backward(dn, n.h, weight, n.rstd, dh=g)
    out = b"".join(v.contiguous().view(torch.uint8).cpu().numpy().tobytes() for v in (y, dx, dw, dweight))
    out += bytes(-len(out) % 4096)
    assert ref.md5_tree(out, 1024).hex() == json.loads(nat.layer_probe(rows, width, seed, 1, 0))["digest"]


@pytest.mark.parametrize("rows,width", [(0, 128), (128, 0), (100, 128), (128, 130), (16512, 128), (128, 32768)])
def test_sizes_it_does_not_take(nat, rows, width):
    r = json.loads(nat.layer_probe(rows, width, 0, 1, 0))
    assert not r["ok"] and "multiples of 128" in r["error"]


def test_the_tool_reports_it(nat):
    from tritonk8ssupervisor_amd.ops import tool

    small = ["--hbm-bytes", str(16 << 20), "--md5-bytes", str(1 << 20), "--copy-bytes", str(16 << 20), "--iters", "1"]
    p = subprocess.run([str(tool("tk8s-probe")), *small, "--layer", "--layer-rows", "512", "--layer-width", "1024"],
                       capture_output=True, text=True, timeout=100)
    r = json.loads(p.stdout)
    assert p.returncode == 0 and r["ok"] and r["layer"]["ok"] and r["layer"]["digest"] == r["layer_expected"]
    assert r["devices"][0]["layer_digest_ok"] == "unpinned" and r["devices"][0]["phase_ms"]["layer"] > 0
    p = subprocess.run([str(tool("tk8s-probe")), *small, "--layer", "--layer-rows", "100"], capture_output=True, text=True, timeout=100)
    r = json.loads(p.stdout)
    assert p.returncode == 1 and not r["ok"] and not r["devices"][0]["ok"]
    p = subprocess.run([str(tool("tk8s-probe")), *small], capture_output=True, text=True, timeout=100)
    assert p.returncode == 0 and "layer" not in json.loads(p.stdout) and "layer" not in json.loads(p.stdout)["devices"][0]["phase_ms"]


@pytest.mark.parametrize("rows,width", [(128, 256), (1152, 1024)])
def test_it_compares_everything_that_a_step_makes(nat, rows, width):
    """Of 12 sampled rows and columns each: h, y and rstd; the norm's 8-bit row with its scales, the gradient's row and
    column, y's and the weight's columns and a tile of the weight, byte for byte; the products; dx and the norm's dw."""
    r = json.loads(nat.layer_probe(rows, width, 3, 1, 0))
    assert r["ok"], r
    blocks = lambda n: n + n // 128  # values and their scales
    assert r["compared"] == {"norm": 12 * (2 * width + 1), "forward": 144, "input_gradient": 144, "weight_gradient": 144,
                             "norm_gradient": 12 * (width + 1),
                             "rounding": 12 * (2 * blocks(width) + 2 * blocks(rows) + blocks(width) + 128 * 128 + 1)}
