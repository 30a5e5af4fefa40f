"""The 8-bit layer without a GPU: its 64-bit oracles against independent statements of the formats,
and what ops/fp8.py and the native launchers refuse before anything is launched."""
from __future__ import annotations

import numpy as np
import pytest

from tritonk8ssupervisor_amd.ops import reference as ref

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def fp8(native_build):
    from tritonk8ssupervisor_amd.ops import fp8

    return fp8


@pytest.fixture(scope="module")
def nat(native_build):
    from tritonk8ssupervisor_amd.ops import native

    return native()


def test_e4m3_table_is_torchs():
    mine = ref.e4m3_values()
    theirs = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(mine, theirs)
    assert mine[0x7E] == 448.0 and mine[1] == 2.0 ** -9


def test_rounding_oracle_agrees_with_torch_on_32_bit_values():
    table = ref.e4m3_values()[:127]
    mid = (table[1:] + table[:-1]) / 2
    v = np.concatenate([table, mid, np.nextafter(mid.astype(np.float32), np.float32(np.inf)),
                        np.nextafter(mid.astype(np.float32), np.float32(-np.inf))]).astype(np.float32)
    v = np.concatenate([v, -v])
    theirs = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(ref.e4m3_bytes(v.astype(np.float64)), theirs)


def test_scale_oracle_is_the_least_power_of_two():
    amax = np.concatenate([448.0 * 2.0 ** np.arange(-100, 100), np.nextafter(448.0 * 2.0 ** np.arange(-100.0, 100), np.inf),
                           np.random.default_rng(1).uniform(1e-6, 1e6, 500)])
    e = ref.e8m0_bytes(amax).astype(int) - 127
    assert (amax <= 448.0 * 2.0 ** e).all() and (amax > 448.0 * 2.0 ** (e - 1.0)).all()
    np.testing.assert_array_equal(ref.e8m0_bytes(np.array([0.0, np.inf, np.nan, 1e-45, 3e38])), [127, 255, 255, 0, 246 + 1])


def test_gradient_oracle_against_differences():
    rng = np.random.default_rng(2)
    h, w, dy, v = rng.normal(size=(5, 33)), rng.normal(size=33), rng.normal(size=(5, 33)), rng.normal(size=(5, 33))
    eps, t = 1e-5, 1e-6
    rstd = ref.rms_norm(h, w, eps)[1]
    dh, dw = ref.rms_norm_backward(dy, h, w, rstd)
    along = ((ref.rms_norm(h + t * v, w, eps)[0] - ref.rms_norm(h - t * v, w, eps)[0]) * dy).sum() / (2 * t)
    assert (dh * v).sum() == pytest.approx(along, rel=1e-7)
    along = ((ref.rms_norm(h, w + t * v[0], eps)[0] - ref.rms_norm(h, w - t * v[0], eps)[0]) * dy).sum() / (2 * t)
    assert (dw * v[0]).sum() == pytest.approx(along, rel=1e-7)


def _operand(rows, cols, tiles=False, ld=None):
    ld = ld or -(-cols // 16) * 16
    sr = -(-rows // 128) if tiles else rows
    values = torch.zeros(rows, ld, dtype=torch.uint8).view(torch.float8_e4m3fn)[:, :cols]
    return values, torch.full((-(-cols // 128), -(-max(sr, 1) // 16) * 16), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu).t()[:sr]


def test_quantize_refuses(fp8):
    x = torch.zeros(4, 256)
    with pytest.raises(ValueError, match="runs on a GPU"):
        fp8.quantize(x)
    with pytest.raises(TypeError, match="must be a tensor"):
        fp8.quantize([[1.0]])
    for bad, what in ((x.double(), "float32, bfloat16 or float16"), (x[0], "2 dimensions"), (x.t(), "contiguous"),
                      (x.to(torch.int32), "float32, bfloat16 or float16")):
        with pytest.raises(ValueError, match=what):
            fp8.quantize(bad)
    with pytest.raises(ValueError, match="layout"):
        fp8.quantize(x, layout="diagonal")


def test_norm_refuses(fp8):
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.ones(256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="runs on a GPU"):
        fp8.rms_norm(x, w)
    for kw, what in (({"residual": x.float()}, "residual must be"), ({"residual": x[:3]}, "residual must be"),
                     ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps")):
        with pytest.raises(ValueError, match=what):
            fp8.rms_norm(x, w, **kw)
    for bad in (w[:255], w.half(), torch.ones(512, dtype=torch.bfloat16)[::2], w[None]):
        with pytest.raises(ValueError, match="weight must be"):
            fp8.rms_norm(x, bad)
    with pytest.raises(TypeError):
        fp8.rms_norm(x, None)


def test_norm_backward_refuses(fp8):
    h, w, r = torch.zeros(4, 256), torch.ones(256), torch.ones(4)
    with pytest.raises(ValueError, match="runs on a GPU"):
        fp8.rms_norm_backward(h, h, w, r)
    for args, what in (((h[:, :128], h, w, r), "dy must be"), ((h.half(), h, w, r), "dy must be"),
                       ((h, h, w, r[:3]), "rstd must be"), ((h, h, w, r.double()), "rstd must be"), ((h, h, w.half(), r), "weight must be")):
        with pytest.raises(ValueError, match=what):
            fp8.rms_norm_backward(*args)
    with pytest.raises(ValueError, match="dh must be"):
        fp8.rms_norm_backward(h, h, w, r, dh=h.half())


def test_matmul_refuses(fp8):
    a, b = _operand(5, 300), _operand(7, 300)
    with pytest.raises(ValueError, match="run"):
        fp8.matmul(a, b)
    with pytest.raises(ValueError, match="run"):
        fp8.matmul(a, _operand(7, 300, tiles=True))
    with pytest.raises(TypeError, match="pair"):
        fp8.matmul(a[0], b[0][0, 0])
    cases = [
        ((a, _operand(7, 299)), "as many columns"),
        ((_operand(5, 300, tiles=True), b), "a's scales must be"),  # 128 x 128 only for b
        (((a[0].float(), a[1]), b), "float8_e4m3fn"),
        (((a[0], a[1].view(torch.uint8)), b), "float8_e8m0fnu"),
        (((a[0], a[1][:, :2]), b), "a's scales must be"),
        ((a, (b[0].contiguous(), b[1])), "16-byte boundaries"),  # rows of 300 bytes
        (((_operand(5, 316)[0][:, 1:301], a[1]), b), "16-byte boundaries"),
    ]
    for args, what in cases:
        with pytest.raises(ValueError, match=what):
            fp8.matmul(*args)
    with pytest.raises(ValueError, match="dtype"):
        fp8.matmul(a, b, dtype=torch.float64)
    for out, what in ((torch.empty(5, 8), "out must be"), (torch.empty(7, 5).t(), "contiguous"),
                      (torch.empty(1, 7).expand(5, 7), "overlap"), (torch.empty(5, 7, dtype=torch.int32), "dtype")):
        with pytest.raises(ValueError, match=what):
            fp8.matmul(a, b, out=out)


def test_native_launchers_refuse_before_launching(nat):
    none = (0, 0, 0, 0)
    with pytest.raises(ValueError, match="type must be"):
        nat.fp8_quantize(4096, 1, 1, 1, 7, none, none, none)
    with pytest.raises(ValueError, match="scales"):
        nat.fp8_quantize(4096, 16, 1, 16, 0, (4096, 16, 0, 0), none, none)
    with pytest.raises(ValueError, match="16-byte"):
        nat.fp8_quantize(4096, 16, 2, 16, 0, (4096, 17, 4096, 16), none, none)
    with pytest.raises(ValueError, match="x is needed"):
        nat.fp8_quantize(0, 16, 2, 16, 0, none, none, none)
    with pytest.raises(ValueError, match="residual needs h"):
        nat.rms_norm_fp8(4096, 16, 4096, 16, 4096, 0, 0, none, 0, 0, 0, 1, 16, 1e-6, 0, 0)
    with pytest.raises(ValueError, match="weight is of"):
        nat.rms_norm_fp8(4096, 16, 0, 0, 4096, 0, 0, none, 0, 0, 0, 1, 16, 1e-6, 0, 1)
    with pytest.raises(ValueError, match="pointer is missing"):
        nat.rms_norm_backward(4096, 16, 4096, 16, 4096, 4096, 0, 0, 0, 16, 4096, 4096, 1, 16, 0, 0)
    assert nat.rms_norm_backward_workspace(1000, 16) > 0  # where one is needed, it is missed
    with pytest.raises(ValueError, match="pointer is missing"):
        nat.rms_norm_backward(4096, 16, 4096, 16, 4096, 4096, 0, 0, 4096, 16, 4096, 0, 1000, 16, 0, 0)
    with pytest.raises(ValueError, match="no rows"):
        nat.rms_norm_backward(4096, 16, 4096, 16, 4096, 4096, 0, 0, 4096, 16, 4096, 4096, 0, 16, 0, 0)
    with pytest.raises(ValueError, match="c is needed"):
        nat.fp8_matmul(none, none, False, 0, 1, 1, 1, 1, 0)
    with pytest.raises(ValueError, match="pointer is missing"):
        nat.fp8_matmul(none, none, False, 4096, 1, 1, 1, 1, 0)
    with pytest.raises(ValueError, match="multiple of 8"):
        nat.layer_fill(4096, 12, 0)
    near, far = (4096, 16, 4096, 1 << 20), (4096, 1 << 23, 4096, 1 << 20)
    for out in (0, 1):
        with pytest.raises(ValueError, match="2\\^34 values"):
            nat.fp8_matmul(near, near, False, 4096, 1 << 20, 1 << 18, 1 << 17, 16, out)
        with pytest.raises(ValueError, match="too many values"):
            nat.fp8_matmul(far, near, False, 4096, 1 << 20, 1 << 17, 1 << 17, 16, out)
    with pytest.raises(ValueError, match="16-byte"):
        nat.fp8_matmul((4096, 17, 4096, 16), (4096, 16, 4096, 16), False, 4096, 1, 1, 1, 1, 0)


def test_matmul_refuses_a_result_that_autograd_would_record(fp8):
    a, b = _operand(5, 300), _operand(7, 300)
    leaf = torch.zeros(5, 7, requires_grad=True)
    with pytest.raises(ValueError, match="requires grad"):
        fp8.matmul(a, b, out=leaf)
    with torch.no_grad(), pytest.raises(ValueError, match="run"):
        fp8.matmul(a, b, out=leaf)


def test_assembly_declares_what_it_writes():
    """The loads to LDS move their address to m0: the compiler has to know."""
    import re
    from pathlib import Path

    sources = Path(__file__).resolve().parents[1] / "native" / "src"
    found = 0
    for f in sources.glob("*.hip"):
        for text in re.findall(r"asm volatile\((.*?)\);", f.read_text(), re.S):
            if "m0" in text.split(":")[0]:
                found += 1
                assert re.search(r':[^:]*"m0"[^:]*$', text), (f.name, text)
    assert found


def test_tensors_that_stand_for_other_values_are_refused(fp8):
    """A lazily negated tensor's memory holds the other sign; zeros may have no memory at all."""
    z = torch.randn(4, 1, dtype=torch.complex64)
    x = z.conj().imag  # rows x 1: its one column is contiguous
    assert x.is_neg()
    w, r = torch.ones(1), torch.ones(4)
    for call in (lambda: fp8.quantize(x), lambda: fp8.rms_norm(x, w), lambda: fp8.rms_norm(torch.ones(4, 1), w, residual=x),
                 lambda: fp8.rms_norm(torch.ones(1, 1), z[0].conj().imag), lambda: fp8.rms_norm_backward(x, torch.ones(4, 1), w, r)):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()
    with pytest.raises(ValueError, match="runs on a GPU"):
        fp8.quantize(x.resolve_neg())
    zeros = torch._efficientzerotensor((4, 1))  # a tangent that autograd never wrote down
    for call in (lambda: fp8.quantize(zeros), lambda: fp8.rms_norm(torch.ones(4, 1), w, residual=zeros),
                 lambda: fp8.rms_norm_backward(torch.ones(4, 1), torch.ones(4, 1), w, r, dh=zeros)):
        with pytest.raises(ValueError, match="without memory"):
            call()
