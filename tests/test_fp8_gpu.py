"""The 8-bit layer's HIP kernels against their 64-bit oracles (ops/reference.py) on a GPU.

Tolerances, derived: one rounding to a type is off by at most half a step (HALF); a 32-bit sum of n
products in any order by at most n * 2^-24 times the sum of their magnitudes. A 16-bit product goes
through the 8-bit matrix instruction, which cuts each of 8 neighbouring products below 2^-13 of the
largest power of two among them: at most 7 * 2^-13 times the largest product of the 8 (the largest
loses nothing). What is rounded to 8 bits has to be equal byte for byte: it is computed from exact
values, or in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from tritonk8ssupervisor_amd.ops import reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in TYPES}  # half the least step


@pytest.fixture(scope="module")
def fp8(native_build):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tritonk8ssupervisor_amd.ops import fp8

    return fp8


def host(t) -> np.ndarray:
    return t.detach().cpu().double().numpy()


def bits(t) -> np.ndarray:
    return t.cpu().view(torch.uint8).numpy()


def close(got: np.ndarray, want: np.ndarray, bound: np.ndarray) -> None:
    off = np.abs(got - want)
    assert got.shape == want.shape
    assert np.isfinite(got).all() and (off <= bound).all(), (off - bound).max()


def randn(seed, *shape, dtype=torch.float32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * spread).to(dtype)


def operand(fp8, seed, rows, cols, tiles=False, spread=1.0):
    """Random bytes of all finite e4m3 values and scales over a wide range, on the GPU as quantize() lays them out."""
    rng = np.random.default_rng(seed)
    q = rng.integers(0, 254, size=(rows, cols)).astype(np.uint8)
    q[(q & 0x7F) == 0x7F] = 0x3A
    sr, nb = (-(-rows // 128) if tiles else rows), -(-cols // 128)
    s = rng.integers(118, 134, size=(sr, nb)).astype(np.uint8)
    values = torch.empty(rows, -(-cols // 16) * 16, dtype=torch.uint8, device="cuda")[:, :cols]
    scales = torch.empty(nb, -(-sr // 16) * 16, dtype=torch.uint8, device="cuda").t()[:sr]
    values.copy_(torch.from_numpy(q))
    scales.copy_(torch.from_numpy(s))
    out = fp8.Quantized(values.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu))
    return out, ref.fp8_dequantize(q, s)


def check_product(c, a64, b64, k):
    want, size = a64 @ b64.T, np.abs(a64) @ np.abs(b64).T
    off = (k + 2) * U * size
    if c.dtype != torch.float32:
        a8, b8 = (np.abs(np.pad(v, ((0, 0), (0, -k % 8)))).reshape(v.shape[0], -1, 8).max(axis=2) for v in (a64, b64))
        off += 7 * 2.0 ** -13 * (a8 @ b8.T)
    got, top = host(c), torch.finfo(c.dtype).max * (1 + HALF[c.dtype] / 2)  # from here on a value rounds to infinity
    over, near = np.abs(want) - off >= top, np.abs(want) + off >= top
    assert (got[over] == np.sign(want[over]) * np.inf).all()
    near &= ~over
    assert (np.isinf(got[near]) | (np.abs(got[near]) <= top)).all()
    fine = ~(over | near)
    close(got[fine], want[fine], (HALF[c.dtype] * (np.abs(want) + off) + TINY[c.dtype] + off)[fine])


# ---- rounding to 8 bits ---------------------------------------------------------------------


def test_rounding_at_every_border(fp8):
    """All e4m3 values, the middles between them and their neighbours, as 32-bit values under scale 1."""
    table = ref.e4m3_values()[:127].astype(np.float32)
    mid = (table[1:] + table[:-1]) / 2
    v = np.concatenate([table, mid, np.nextafter(mid, np.float32(np.inf)), np.nextafter(mid, np.float32(-np.inf))])
    v = np.concatenate([v, -v])
    x = np.zeros((8, 128), dtype=np.float32)
    x[:, 0] = 448.0
    x[:, 1:].flat[: v.size] = v
    x = np.concatenate([x, np.pad(v, (0, -v.size % 127)).reshape(-1, 127) @ np.eye(127, 128, 1, dtype=np.float32)])
    x[8:, 0] = 448.0
    q, s = fp8.quantize(torch.from_numpy(x).cuda())
    want, scales = ref.fp8_quantize(x.astype(np.float64))
    assert (scales == 127).all()
    np.testing.assert_array_equal(bits(s), scales)
    got, neg0 = bits(q), want == 0x80
    np.testing.assert_array_equal(np.where(neg0, 0x80, got), want)


def test_scales_at_their_borders(fp8):
    tops = np.array([448.0 * 2.0 ** e for e in (-130, -120, -30, -1, 0, 1, 60, 118, 119)], dtype=np.float32)
    tops = np.concatenate([tops, np.nextafter(tops[1:-1], np.float32(np.inf)), np.float32([0.0, 1e-45, 1e-40, 3.4e38])])
    x = np.zeros((tops.size, 256), dtype=np.float32)
    x[:, 3], x[:, 200] = -tops, tops / 3
    x[:, 7] = tops * np.float32(0.37)
    q, s = fp8.quantize(torch.from_numpy(x).cuda())
    want, scales = ref.fp8_quantize(x.astype(np.float64))
    np.testing.assert_array_equal(bits(s), scales)
    np.testing.assert_array_equal(host(q), ref.e4m3_values()[want])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_block_that_is_not_finite_is_nan_and_its_neighbours_are_not(fp8, bad):
    x = randn(3, 130, 300, dtype=torch.bfloat16)
    x[5, 140] = bad
    (q, s), (qt, st) = fp8.quantize(x.cuda(), layout="both")
    tiles = fp8.quantize(x.cuda(), layout="tiles")
    for (v, sc), rows, cols in (((q, s), slice(5, 6), slice(128, 256)), ((qt, st), slice(140, 141), slice(0, 128)),
                                (tiles, slice(0, 128), slice(128, 256))):
        v = host(v)
        assert np.isnan(v[rows, cols]).all()
        v[rows, cols] = 0
        assert not np.isnan(v).any()
        assert (bits(sc) == 255).sum() == 1


@pytest.mark.parametrize("layout", ["rows", "columns", "both", "tiles"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 127), (129, 130), (128, 128), (257, 1000), (16, 33), (1000, 7)])
def test_quantize_matches_the_oracle(fp8, layout, dtype, rows, cols):
    x = randn(rows * cols, rows, cols, dtype=dtype) * torch.exp2(torch.arange(rows) % 9 - 6.0)[:, None].to(dtype)
    x[rows // 2] = 0
    out = fp8.quantize(x.cuda(), layout=layout)
    x64 = x.double().numpy()
    for (q, s), want in zip(out if layout == "both" else (out,), {
            "rows": [(x64, 1)], "columns": [(x64.T, 1)], "both": [(x64, 1), (x64.T, 1)], "tiles": [(x64, 128)]}[layout]):
        values, scales = ref.fp8_quantize(*want)
        np.testing.assert_array_equal(bits(s), scales)
        np.testing.assert_array_equal(host(q), ref.e4m3_values()[values])


def test_quantize_takes_strided_rows_and_leaves_what_is_behind_them(fp8):
    """Rows of a wider matrix that start at an odd place; the padding of the outputs stays as it was."""
    wide = randn(4, 70, 301, dtype=torch.bfloat16).cuda()
    x = wide[3:60, 5:206]
    for layout in ("rows", "columns", "tiles"):
        got, want = fp8.quantize(x, layout=layout), fp8.quantize(x.contiguous(), layout=layout)
        np.testing.assert_array_equal(bits(got.values.contiguous()), bits(want.values.contiguous()))
        np.testing.assert_array_equal(bits(got.scales.contiguous()), bits(want.scales.contiguous()))
    from tritonk8ssupervisor_amd.ops import native

    rows, cols, ld = x.shape[0], x.shape[1], 224
    q = torch.full((rows + 2, ld), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((3, 64), 0x55, dtype=torch.uint8, device="cuda")
    t = torch.full((cols + 2, 64), 0x55, dtype=torch.uint8, device="cuda")
    st = torch.full((2, 224), 0x55, dtype=torch.uint8, device="cuda")
    native().fp8_quantize(x.data_ptr(), x.stride(0), rows, cols, 1, (q.data_ptr(), ld, s.data_ptr(), 64),
                          (t.data_ptr(), 64, st.data_ptr(), 224), (0, 0, 0, 0), torch.cuda.current_stream().cuda_stream)
    assert (q[rows:] == 0x55).all() and (q[:, cols:] == 0x55).all()
    assert (s[2:] == 0x55).all() and (s[:, rows:] == 0x55).all()
    assert (t[cols:] == 0x55).all() and (t[:, rows:] == 0x55).all()
    assert (st[1:] == 0x55).all() and (st[:, cols:] == 0x55).all()


def test_quantize_of_nothing(fp8):
    for shape in ((0, 256), (5, 0)):
        x = torch.empty(shape, device="cuda")
        assert fp8.quantize(x).values.shape == shape
        assert fp8.quantize(x, layout="columns").values.shape == shape[::-1]
        assert fp8.quantize(x, layout="tiles").values.shape == shape


# ---- norm ---------------------------------------------------------------------------------


NORM_SHAPES = [(1, 1), (1, 4096), (2, 127), (5, 512), (4, 513), (7, 1024), (3, 1100), (3, 2048), (6, 2049), (2, 5003), (3, 8192),
               (2, 8200), (2, 16384), (2, 16400), (3, 40000), (300, 136)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_norm_matches_the_oracle(fp8, dtype, residual, rows, cols):
    x = randn(rows + cols, rows, cols, dtype=dtype, spread=3.0)
    r = randn(7, rows, cols, dtype=dtype) if residual else None
    wide = dtype != torch.float32 and cols % 2 == 0  # a 32-bit weight beside 16-bit values
    w = (1.0 + randn(5, cols, spread=0.2)).to(torch.float32 if wide else dtype)
    if rows > 2:
        x[1] = 0
        if residual:
            r[1] = 0  # a row of zeros: rstd is 1 / sqrt(eps), y is 0
    eps = 1e-5
    n = fp8.rms_norm(x.cuda(), w.cuda(), residual=None if r is None else r.cuda(), eps=eps, normed=True)
    h = x if r is None else (x.float() + r.float()).to(dtype)
    assert torch.equal(n.h.cpu(), h)
    y, rstd = ref.rms_norm(h.double().numpy(), w.double().numpy(), eps)
    q, s = ref.fp8_quantize(y)
    np.testing.assert_array_equal(bits(n.scales), s)
    np.testing.assert_array_equal(host(n.values), ref.e4m3_values()[q])
    close(host(n.rstd), rstd, 1.0001 * U * rstd)
    close(host(n.y), y, 1.0001 * HALF[dtype] * np.abs(y) + TINY[dtype])
    only = fp8.rms_norm(x.cuda(), w.cuda(), residual=None if r is None else r.cuda(), eps=eps, quantized=False, normed=True)
    assert only.values is None and torch.equal(only.y, n.y)


def test_norm_of_rows_that_are_not_finite(fp8):
    x = randn(1, 6, 700, dtype=torch.bfloat16)
    x[1, 3], x[3, 650] = float("nan"), float("inf")
    w = torch.ones(700, dtype=torch.bfloat16)
    n = fp8.rms_norm(x.cuda(), w.cuda(), normed=True)
    y, _ = ref.rms_norm(x.double().numpy(), w.double().numpy(), 1e-6)
    q, s = ref.fp8_quantize(y)
    np.testing.assert_array_equal(bits(n.scales), s)
    np.testing.assert_array_equal(np.isnan(host(n.values)), np.isnan(ref.e4m3_values()[q]))
    ok = [0, 2, 4, 5]
    np.testing.assert_array_equal(host(n.values)[ok], ref.e4m3_values()[q][ok])
    assert np.isnan(host(n.values)[1]).all()  # the sum is NaN; an infinity: 0 elsewhere, NaN where it stands
    assert (host(n.values)[3, :512] == 0).all() and np.isnan(host(n.values)[3, 640:]).all()


def test_norm_takes_strided_rows(fp8):
    wide = randn(2, 9, 5000, dtype=torch.float16).cuda()
    x, r = wide[1:6, 3:1504], wide[3:8, 1600:3101]
    w = (1.0 + randn(5, 1501, spread=0.2)).half().cuda()
    got, want = fp8.rms_norm(x, w, residual=r), fp8.rms_norm(x.contiguous(), w, residual=r.contiguous())
    assert torch.equal(got.h, want.h)
    np.testing.assert_array_equal(bits(got.values.contiguous()), bits(want.values.contiguous()))
    np.testing.assert_array_equal(bits(got.scales.contiguous()), bits(want.scales.contiguous()))


def test_norm_of_nothing(fp8):
    n = fp8.rms_norm(torch.empty(0, 256, device="cuda"), torch.ones(256, device="cuda"))
    assert n.values.shape == (0, 256) and n.scales.shape == (0, 2) and n.rstd.shape == (0,)
    dx, dw = fp8.rms_norm_backward(n.h, n.h, torch.ones(256, device="cuda"), n.rstd)
    assert dx.shape == (0, 256) and (dw == 0).all()


# ---- the norm's gradient ----------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("more", [False, True])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES + [(1500, 260), (1025, 17), (2500, 126), (700, 250), (1100, 1003), (600, 437), (1026, 2047), (515, 4098), (9000, 129), (9000, 2404), (17000, 2100)])
def test_norm_backward_matches_the_oracle(fp8, dtype, more, rows, cols):
    h = randn(rows + cols, rows, cols, dtype=dtype, spread=2.0)
    dy = randn(8, rows, cols, dtype=dtype)
    dh = randn(9, rows, cols, dtype=dtype) if more else None
    w = (1.0 + randn(5, cols, spread=0.2)).to(dtype)
    rstd = (1.0 / torch.sqrt(h.double().square().mean(1) + 1e-5)).float()
    dx, dw = fp8.rms_norm_backward(dy.cuda(), h.cuda(), w.cuda(), rstd.cuda(), dh=None if dh is None else dh.cuda())
    h64, dy64, w64, r64 = (t.double().numpy() for t in (h, dy, w, rstd))
    dx64, dw64 = ref.rms_norm_backward(dy64, h64, w64, r64)
    extra = 0.0 if dh is None else dh.double().numpy()
    xh, g = h64 * r64[:, None], dy64 * w64
    # g, xh, their products, the sum over the row, the mean, its product with xh, the difference, times rstd, plus dh
    mean = np.abs(g * xh).mean(axis=1, keepdims=True)
    size = r64[:, None] * (4 * np.abs(g) + np.abs(xh) * mean * (cols + 8)) + 2 * np.abs(extra)
    close(host(dx), dx64 + extra, HALF[dtype] * np.abs(dx64 + extra) + TINY[dtype] + 1.01 * U * size)
    close(host(dw), dw64, (rows + 4) * U * np.abs(dy64 * xh).sum(axis=0) + TINY[torch.float32])


def test_norm_backward_against_differences(fp8):
    """The GPU's gradients along random directions against the change of sum(dy * y) in 64 bits."""
    h, dy, v = (randn(s, 6, 777, dtype=torch.float32) for s in (1, 2, 3))
    w, vw = 1.0 + randn(4, 777, spread=0.2), randn(5, 777)
    eps, t = 1e-5, 1e-5
    rstd = fp8.rms_norm(h.cuda(), w.cuda(), eps=eps).rstd
    dx, dw = fp8.rms_norm_backward(dy.cuda(), h.cuda(), w.cuda(), rstd)
    h, dy, v, w, vw = (x.double().numpy() for x in (h, dy, v, w, vw))

    def change(h1, w1, h2, w2):
        return ((ref.rms_norm(h1, w1, eps)[0] - ref.rms_norm(h2, w2, eps)[0]) * dy).sum() / (2 * t)

    along_h, along_w = change(h + t * v, w, h - t * v, w), change(h, w + t * vw, h, w - t * vw)
    assert abs((host(dx) * v).sum() - along_h) <= 1e-5 * np.abs(host(dx) * v).sum()
    assert abs((host(dw) * vw).sum() - along_w) <= 1e-5 * np.abs(host(dw) * vw).sum()


# ---- product --------------------------------------------------------------------------------


SIZES = [(3, 1500, 700), (5, 9000, 260), (20, 14400, 520), (33, 4100, 1500), (130, 8200, 400), (64, 6200, 2100), (50, 6300, 1000), (8, 6150, 200), (20, 6400, 1100), (40, 6200, 130), (64, 700, 3000), (70, 64, 512), (97, 450, 2049), (1, 1, 1), (1, 16, 128), (1, 4096, 512), (2, 130, 300), (7, 100, 1000), (16, 64, 127), (17, 129, 129), (33, 257, 640),
         (64, 64, 64), (65, 300, 4100), (128, 128, 128), (129, 1, 257), (200, 333, 17), (256, 256, 256), (300, 520, 1030),
         (513, 257, 384), (1, 7, 20000), (31, 40, 9000)]


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul_matches_the_oracle(fp8, m, n, k, tiles, out):
    a, a64 = operand(fp8, m + k, m, k)
    b, b64 = operand(fp8, n + 2 * k, n, k, tiles=tiles)
    if out == torch.float16:  # within its range
        a64 = a64 * 2.0 ** -14
        a.scales.view(torch.uint8).sub_(14)
    check_product(fp8.matmul(a, b, dtype=out), a64, b64, k)


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("m,n,k", [(3621, 3700, 128), (3600, 3585, 300), (3585, 3612, 640), (3584, 3584, 1029)])
def test_matmul_of_many_tiles_matches_the_oracle(fp8, m, n, k, tiles):
    """Enough of C for the largest tiles, cut off at every side; 1 to 8 blocks of k."""
    a, a64 = operand(fp8, m + k, m, k)
    b, b64 = operand(fp8, n + 2 * k, n, k, tiles=tiles)
    out = torch.full((m + 1, n + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    check_product(fp8.matmul(a, b, out=out[:m, 3:3 + n]), a64, b64, k)
    assert (out[m:] == 7).all() and (out[:, :3] == 7).all() and (out[:, 3 + n:] == 7).all()


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("m,n,k", [(1100, 1190, 513), (1990, 2003, 300), (2050, 1921, 1024), (2100, 2113, 640), (2177, 2050, 1029), (2900, 2055, 400)])
def test_matmul_of_some_tiles_matches_the_oracle(fp8, m, n, k, tiles, out):
    """Between few rows and many tiles, cut off at every side; NaN and the largest scale behind the operands."""
    a, a64 = operand(fp8, m + k, m, k)
    b, b64 = operand(fp8, n + 2 * k, n, k, tiles=tiles)

    def buried(q):
        rows, ld, blocks = q.values.shape[0], -(-k // 16) * 16 + 16, q.scales.shape[1]
        v = torch.full((rows + 3, ld), 0x7F, dtype=torch.uint8, device="cuda")
        v[:rows, :k] = q.values.view(torch.uint8)
        s = torch.full((blocks + 1, -(-q.scales.shape[0] // 4) * 4 + 4), 255, dtype=torch.uint8, device="cuda")
        s[:blocks, :q.scales.shape[0]] = q.scales.view(torch.uint8).t()
        return fp8.Quantized(v.view(torch.float8_e4m3fn)[:rows, :k], s.view(torch.float8_e8m0fnu).t()[:q.scales.shape[0], :blocks])

    c = torch.full((m + 1, n + 8), 7.0, dtype=out, device="cuda")
    got = fp8.matmul(buried(a), buried(b), out=c[:m, 3:3 + n])
    check_product(got, a64, b64, k)
    assert (c[m:] == 7).all() and (c[:, :3] == 7).all() and (c[:, 3 + n:] == 7).all()
    assert torch.equal(fp8.matmul(a, b, dtype=out), got)
    a.values.view(torch.uint8)[m - 2, k - 1] = 0x7F
    b.scales.view(torch.uint8)[-1, -1] = 255
    if not tiles:
        bad = fp8.matmul(a, b, dtype=out).isnan()
        assert bad[m - 2].all() and bad[:, n - 1].all() and bad.sum() == m + n - 1


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(2000, 2000), (2100, 2100), (2900, 2100), (3600, 3600)])
def test_matmul_of_more_tiles_at_the_ends_of_the_scales(fp8, m, n, out):
    a, _ = operand(fp8, 1, m, 300)
    b, _ = operand(fp8, 2, n, 300)
    a.values.view(torch.uint8).fill_(0x38)  # ones
    b.values.view(torch.uint8).fill_(0x38)
    for sa, sb, want in ((0, 254, 300.0), (254, 0, 300.0), (0, 200, 300.0 * 2.0 ** -54), (254, 127, np.inf), (27, 227, 300.0)):
        a.scales.view(torch.uint8).fill_(127)
        b.scales.view(torch.uint8).fill_(127)
        a.scales.view(torch.uint8)[1000:].fill_(sa)  # far ones in the later tiles alone
        b.scales.view(torch.uint8)[900:].fill_(sb)
        c = host(fp8.matmul(a, b, dtype=out))
        want = host(torch.tensor([want]).to(out))
        assert (c[:1000, :900] == host(torch.tensor([300.0]).to(out))).all() and (c[1000:, 900:] == want).all(), (sa, sb)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_matmul_of_rows_far_apart(fp8, out):
    """Rows 2^23 bytes apart: offsets into A pass 32 bits."""
    m, n, k = 600, 70, 300
    a, a64 = operand(fp8, 1, m, k)
    b, b64 = operand(fp8, 2, n, k)
    far = torch.empty(m, 1 << 23, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    far[:, :k].view(torch.uint8).copy_(a.values.view(torch.uint8))
    got = fp8.matmul((far[:, :k], a.scales), b, dtype=out)
    check_product(got, a64, b64, k)
    check_product(fp8.matmul(b, (far[:, :k], a.scales), dtype=out), b64, a64, k)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [1, 16, 100, 127])
def test_matmul_of_less_than_a_block(fp8, k, out):
    """However large C is."""
    for m, n in ((3, 2050), (600, 700), (1500, 1500), (3600, 3600)):
        a, a64 = operand(fp8, m, m, k)
        b, b64 = operand(fp8, n + 1, n, k)
        check_product(fp8.matmul(a, b, dtype=out), a64, b64, k)


def test_matmul_of_whole_numbers_is_exact(fp8):
    """Small whole numbers: every product and sum is a 32-bit value, so nothing may be off."""
    rng = np.random.default_rng(5)
    for m, n, k in ((3, 200, 1000), (300, 270, 1100), (2000, 2100, 1100)):
        x, y = rng.integers(-8, 9, (m, k)), rng.integers(-8, 9, (n, k))
        a, b = (fp8.quantize(torch.from_numpy(z).float().cuda()) for z in (x, y))
        np.testing.assert_array_equal(host(fp8.matmul(a, b, dtype=torch.float32)), x @ y.T)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [20, 150])
def test_matmul_at_the_ends_of_the_scales(fp8, m, out):
    """2^-127 and 2^127 against each other, and sums near both ends of what 32 bits hold."""
    a, _ = operand(fp8, 1, m, 256)
    b, _ = operand(fp8, 2, 24, 256)
    a.values.view(torch.uint8).fill_(0x38)  # ones
    b.values.view(torch.uint8).fill_(0x38)
    for sa, sb, want in ((0, 254, 256.0), (254, 0, 256.0), (127, 0, 256.0 * 2.0 ** -127), (0, 200, 256.0 * 2.0 ** -54),
                         (254, 127, np.inf), (254, 112, 256.0 * 2.0 ** 112), (27, 227, 256.0), (28, 226, 256.0)):
        a.scales.view(torch.uint8).fill_(sa)
        b.scales.view(torch.uint8).fill_(sb)
        c = host(fp8.matmul(a, b, dtype=out))
        assert (c == want).all(), (sa, sb, c[0, 0], want)


def test_matmul_takes_scales_that_lie_row_by_row(fp8):
    a, a64 = operand(fp8, 1, 70, 400)
    b, b64 = operand(fp8, 2, 90, 400)
    want = fp8.matmul(a, b)
    check_product(want, a64, b64, 400)
    assert torch.equal(fp8.matmul((a.values, a.scales.contiguous()), (b.values, b.scales.contiguous())), want)
    odd = torch.empty(4, 73, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu).t()[1:71]  # no dword starts a block
    assert torch.equal(fp8.matmul((a.values, odd.copy_(a.scales)), b), want)
    one = fp8.matmul((a.values[:1], a.scales[:1]), b)
    assert torch.equal(one, want[:1])


def test_matmul_carries_nan_to_its_row_and_column_alone(fp8):
    a, _ = operand(fp8, 1, 200, 400)
    b, _ = operand(fp8, 2, 300, 400)
    a.values.view(torch.uint8)[17, 399] = 0x7F
    b.scales.view(torch.uint8)[250, 1] = 255
    for m, out in ((200, torch.float32), (200, torch.bfloat16), (18, torch.float32), (18, torch.bfloat16)):
        c = host(fp8.matmul((a.values[:m], a.scales[:m]), b, dtype=out))
        nan = np.zeros((m, 300), dtype=bool)
        nan[17], nan[:, 250] = True, True
        np.testing.assert_array_equal(np.isnan(c), nan)


@pytest.mark.parametrize("m", [1, 30, 150])
def test_matmul_reads_nothing_behind_its_operands(fp8, m):
    """NaN in the rows' padding, behind the last row and in the scales of rows that are not there."""
    k, n = 300, 70
    a, a64 = operand(fp8, 3, m, k)
    b, b64 = operand(fp8, 4, n, k)

    def buried(q, rows):
        ld = 336
        v = torch.full((rows + 3, ld), 0x7F, dtype=torch.uint8, device="cuda")
        v[:rows, :k] = q.values.view(torch.uint8)
        s = torch.full((4, 176), 255, dtype=torch.uint8, device="cuda")
        s[:3, :rows] = q.scales.view(torch.uint8).t()
        return fp8.Quantized(v.view(torch.float8_e4m3fn)[:rows, :k], s.view(torch.float8_e8m0fnu).t()[:rows, :3])

    want = fp8.matmul(a, b)
    out = torch.full((m + 2, n + 5), 7.0, dtype=torch.bfloat16, device="cuda")
    got = fp8.matmul(buried(a, m), buried(b, n), out=out[:m, 2:2 + n])
    assert torch.equal(got, want)
    assert (out[m:] == 7).all() and (out[:, :2] == 7).all() and (out[:, 2 + n:] == 7).all()
    check_product(want, a64, b64, k)


def test_matmul_of_nothing(fp8):
    a, _ = operand(fp8, 1, 5, 0)
    b, _ = operand(fp8, 1, 7, 0)
    assert (fp8.matmul(a, b) == 0).all()
    a, _ = operand(fp8, 1, 0, 256)
    b, _ = operand(fp8, 1, 7, 256)
    assert fp8.matmul(a, b).shape == (0, 7) and fp8.matmul(b, a).shape == (7, 0)


# ---- together, on streams, in graphs -----------------------------------------------------------


def layer(fp8, x, residual, norm_weight, w, wt, dout, dh):
    """One layer forward and backward as a program runs it."""
    n = fp8.rms_norm(x, norm_weight, residual=residual, normed=True)
    out = fp8.matmul(n.quantized, w)
    drows, dcols = fp8.quantize(dout, layout="both")
    dy = fp8.matmul(drows, wt)
    dw = fp8.matmul(dcols, fp8.quantize(n.y, layout="columns"), dtype=torch.float32)
    dx, dnorm = fp8.rms_norm_backward(dy, n.h, norm_weight, n.rstd, dh=dh)
    return {"h": n.h, "out": out, "dw": dw, "dx": dx, "dnorm": dnorm, "dy": dy}


def layer_inputs(fp8, tokens, width, wide, seed=0):
    x, r, dh = (randn(seed + s, tokens, width, dtype=torch.bfloat16).cuda() for s in (1, 2, 6))
    weight = (randn(seed + 3, wide, width) * width ** -0.5).cuda()
    norm_weight = (1.0 + randn(seed + 4, width, spread=0.2)).bfloat16().cuda()
    dout = (randn(seed + 5, tokens, wide) * 1e-3).bfloat16().cuda()
    return (x, r, norm_weight, fp8.quantize(weight, layout="tiles"), fp8.quantize(weight.t().contiguous(), layout="tiles"), dout, dh)


@pytest.mark.parametrize("tokens,width,wide", [(1, 512, 640), (203, 520, 300), (300, 1000, 1152)])
def test_a_layer_forward_and_backward(fp8, tokens, width, wide):
    args = layer_inputs(fp8, tokens, width, wide)
    x, r, nw, w, wt, dout, dh = args
    got = layer(fp8, *args)
    h = (x.float() + r.float()).bfloat16().cpu().double().numpy()
    y, rstd = ref.rms_norm(h, host(nw), 1e-6)
    yq = ref.fp8_dequantize(*ref.fp8_quantize(y))
    w64 = ref.fp8_dequantize(bits(w.values.contiguous()), bits(w.scales.contiguous()))
    wt64 = ref.fp8_dequantize(bits(wt.values.contiguous()), bits(wt.scales.contiguous()))
    np.testing.assert_array_equal(wt64, w64.T)  # tiles of a transpose are the tiles' transposes
    check_product(got["out"], yq, w64, width)
    d64 = host(dout)
    dq = ref.fp8_dequantize(*ref.fp8_quantize(d64))
    check_product(got["dy"], dq, wt64, wide)
    y16 = host(fp8.rms_norm(x, nw, residual=r, normed=True).y)
    check_product(got["dw"], ref.fp8_dequantize(*ref.fp8_quantize(d64.T)), ref.fp8_dequantize(*ref.fp8_quantize(y16.T)), tokens)
    dx64, dn64 = ref.rms_norm_backward(host(got["dy"]), h, host(nw), rstd)
    want = dx64 + host(dh)
    xh, g = h * rstd[:, None], host(got["dy"]) * host(nw)
    size = rstd[:, None] * (4 * np.abs(g) + np.abs(xh) * np.abs(g * xh).mean(axis=1, keepdims=True) * (width + 12)) + 2 * np.abs(host(dh))
    close(host(got["dx"]), want, HALF[torch.bfloat16] * np.abs(want) + 2 * U * size)
    close(host(got["dnorm"]), dn64, (tokens + 8) * U * np.abs(host(got["dy"]) * xh).sum(axis=0))
    again = layer(fp8, *args)
    for key in got:
        assert torch.equal(got[key], again[key]), key


def test_a_layer_in_a_graph_replayed(fp8):
    """Captured once, replayed with new inputs between eager runs of other sizes and synchronizations."""
    args = layer_inputs(fp8, 203, 520, 300)
    layer(fp8, *args)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), layer_inputs(fp8, 77, 640, 512, seed=50)
    with torch.cuda.graph(graph):
        captured = layer(fp8, *args)
    for turn in range(4):
        fresh = layer_inputs(fp8, 203, 520, 300, seed=100 * turn)
        for to, new in zip(args, fresh):
            for t, s in zip(to, new) if isinstance(to, tuple) else ((to, new),):
                t.copy_(s)
        layer(fp8, *other)
        graph.replay()
        torch.cuda.synchronize()
        eager = layer(fp8, *fresh)
        for key in eager:
            assert torch.equal(captured[key], eager[key]), (turn, key)


def test_two_streams_at_once(fp8):
    inputs = [layer_inputs(fp8, 300, 1000, 1152, seed=s) for s in (0, 50)]
    want = [layer(fp8, *i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(layer(fp8, *inputs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for run in got[k]:
            for key in run:
                assert torch.equal(run[key], want[k][key]), (k, key)


def test_more_values_than_32_bits_count(fp8):
    """2.3e9 values: the last rows come out as they do by themselves."""
    rows, cols, tail = 70000, 32768, 112  # 70000 = 546 * 128 + 112
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x.view(torch.int16).copy_(torch.arange(cols, dtype=torch.int16, device="cuda") % 199 + 16100)
    x[-tail:].mul_(torch.randn(tail, 1, device="cuda").bfloat16()).add_(torch.randn(tail, cols, device="cuda").bfloat16())
    end = x[-tail:].clone()
    for layout in ("rows", "both", "tiles"):
        whole, part = fp8.quantize(x, layout=layout), fp8.quantize(end, layout=layout)
        if layout == "both":
            assert torch.equal(bits_of(whole[1].values[:, -tail:]), bits_of(part[1].values))
            assert torch.equal(bits_of(whole[1].scales[:, -1]), bits_of(part[1].scales[:, -1]))
            whole, part = whole[0], part[0]
        assert torch.equal(bits_of(whole.values[-tail:]), bits_of(part.values)), layout
        n = 1 if layout == "tiles" else tail
        assert torch.equal(bits_of(whole.scales[-n:]), bits_of(part.scales[-n:])), layout
        del whole, part
    w = torch.randn(cols, device="cuda").bfloat16()
    whole, part = fp8.rms_norm(x, w, normed=True), fp8.rms_norm(end, w, normed=True)
    assert torch.equal(bits_of(whole.values[-tail:]), bits_of(part.values)) and torch.equal(whole.y[-tail:], part.y)
    assert torch.equal(bits_of(whole.scales[-tail:]), bits_of(part.scales)) and torch.equal(whole.rstd[-tail:], part.rstd)
    rstd = whole.rstd
    del whole
    dx, dw = fp8.rms_norm_backward(x, x, w, rstd)
    dx1, _ = fp8.rms_norm_backward(end, end, w, part.rstd)
    assert torch.equal(dx[-tail:], dx1)
    want = sum((x[i:i + 5000].double().square() * rstd[i:i + 5000, None].double()).sum(0) for i in range(0, rows, 5000))
    assert ((dw.double() - want).abs() <= (rows + 8) * U * want).all()


def bits_of(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("m,n", [((1 << 21) + 5, 2100), (70, (1 << 24) + 9)])
def test_products_of_more_values_than_32_bits_count(fp8, m, n):
    k = 130
    def rows_of(seed, rows):
        small, small64 = operand(fp8, seed, 512, k)
        i = torch.arange(rows, device="cuda") % 509
        return fp8.Quantized(torch.nn.functional.pad(bits_of(small.values), (0, 14))[i].view(torch.float8_e4m3fn)[:, :k],
                             bits_of(small.scales).t()[:, i].contiguous().view(torch.float8_e8m0fnu).t()), small64
    (a, a64), (b, b64) = rows_of(1, m), rows_of(2, n)
    c = fp8.matmul(a, b)
    for r, q in ((slice(0, 70), slice(0, 300)), (slice(m - 70, m), slice(n - 300, n)), (slice(m // 2, m // 2 + 64), slice(n // 2, n // 2 + 99))):
        check_product(c[r, q], a64[np.arange(m)[r] % 509], b64[np.arange(n)[q] % 509], k)


@pytest.mark.parametrize("cols", [200, 4096, 40000])
def test_what_a_call_returns_does_not_overlap(fp8, cols):
    """Small results share an allocation: writing to one leaves the others."""
    x, w = torch.randn(3, cols, device="cuda"), torch.randn(cols, device="cuda")
    n = fp8.rms_norm(x, w, residual=x, normed=True)
    results = {"norm": [n.h, n.values, n.scales, n.y, n.rstd], "both": [t for q in fp8.quantize(x, layout="both") for t in q],
               "tiles": list(fp8.quantize(x, layout="tiles")), "backward": list(fp8.rms_norm_backward(x, n.h, w, n.rstd))}
    for name, got in results.items():
        want = [bits_of(t).clone() for t in got]
        for i, t in enumerate(got):
            (t if t.dtype == torch.float32 else t.view(torch.uint8)).fill_(85)
            for j, u in enumerate(got):
                assert j <= i or torch.equal(bits_of(u), want[j]), (name, i, j)


# ---- ends of ranges, and what torch may do with arguments and results ----------------------------


@pytest.mark.parametrize("rows", [5, 30000])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_of_no_columns(fp8, rows, residual):
    """The mean of nothing is NaN and so is rstd, whatever the memory held before."""
    for dtype in TYPES:
        held = [torch.full((rows,), 7.0, device="cuda") for _ in range(4)]
        del held
        x, w = torch.empty(rows, 0, dtype=dtype, device="cuda"), torch.empty(0, dtype=dtype, device="cuda")
        n = fp8.rms_norm(x, w, residual=x if residual else None, normed=True)
        assert n.values.shape == n.y.shape == n.h.shape == (rows, 0) and n.scales.shape == (rows, 0)
        assert n.rstd.shape == (rows,) and n.rstd.isnan().all()


def tiny_case(name):
    """(x, weight, eps) whose products, results or rstd leave the normal numbers of 32 bits."""
    g = np.random.default_rng(11)
    x, w = g.normal(size=(64, 17000)), np.exp2(g.uniform(-1, 1, 17000))
    if name == "tiny products":  # h w is subnormal, y is not
        return x * 1e-3, w * 1.5e-38, 1e-12
    if name == "vanishing products":  # h w is 0 in 32 bits
        return x * 1e-12, w * 1e-36, 1e-28
    if name == "tiny results":
        return x, w * 1e-39, 1e-6
    if name == "tiny products beside large ones":  # blocks of either kind in one wave
        return x * 1e-3, np.where(np.arange(17000) // 128 % 2 == 0, w, w * 1.5e-38), 1e-12
    if name == "tiny rstd":
        return x * 3e37, w * 1e-3, 1e-6
    if name == "small rows":  # rstd is beyond 32 bits
        return x * 1e-39, w, 0.0
    assert name == "tiny rows"
    return x * 1e-41, w, 0.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1000, 104, 200, 600, 17000])
@pytest.mark.parametrize("name", ["tiny products", "vanishing products", "tiny results", "tiny products beside large ones", "tiny rstd", "small rows", "tiny rows"])
def test_norm_at_the_ends_of_32_bits(fp8, name, cols, dtype):
    x, w, eps = tiny_case(name)
    x, w = torch.from_numpy(x[:, :cols].copy()).to(dtype), torch.from_numpy(w[:cols].copy())
    w = w.to(torch.float32 if dtype == torch.float16 else dtype)
    x[3], x[5, 7:20] = 0, 0
    n = fp8.rms_norm(x.cuda(), w.cuda(), eps=eps)
    with np.errstate(divide="ignore", invalid="ignore"):  # a row of zeros whose eps is 0 is NaN
        y, _ = ref.rms_norm(x.double().numpy(), w.double().numpy(), eps)
    q, s = ref.fp8_quantize(y)
    np.testing.assert_array_equal(bits(n.scales), s)
    np.testing.assert_array_equal(host(n.values), ref.e4m3_values()[q])
    rows = np.isfinite(y).all(axis=1)
    full = fp8.rms_norm(x.cuda(), w.cuda(), eps=eps, normed=True)
    np.testing.assert_array_equal(bits(full.values), bits(n.values))
    close(host(full.y)[rows], y[rows], 1.0001 * HALF[dtype] * np.abs(y[rows]) + 1.0001 * TINY[dtype])


def test_norm_backward_of_rows_that_fill_a_launch(fp8):
    """2^27 columns and some: 32 columns to a block of 1024 threads would be 2^32 threads."""
    rows, cols = 2, (1 << 27) + 40
    i = torch.arange(cols, device="cuda")
    h = torch.stack([i % 251 - 125, i % 127 - 63]).bfloat16()
    dy = torch.stack([i % 61 - 30, i % 113 - 56]).bfloat16()
    w, rstd = (i % 5 + 1).bfloat16(), torch.tensor([0.5, 0.25], device="cuda")
    dx, dw = fp8.rms_norm_backward(dy, h, w, rstd)
    want = (dy.float() * h.float() * rstd[:, None]).sum(0)  # every product and sum is exact in 32 bits
    assert torch.equal(dw, want)
    del want
    part = slice(cols - 1000, cols)
    mean = torch.stack([(dy[r].float() * w.float() * h[r].float()).sum(dtype=torch.float64) * rstd[r] / cols for r in range(rows)])
    g, xh = (dy[:, part].double() * w[part].double()), h[:, part].double() * rstd[:, None]
    want = rstd[:, None] * (g - xh * mean[:, None])
    size = rstd[:, None] * (4 * g.abs() + xh.abs() * 30 * 5 * 63)  # a sum over 2^27 in 1024 threads: (2^17 + 30) roundings of the mean's parts
    assert ((dx[:, part].double() - want).abs() <= HALF[torch.bfloat16] * want.abs() + (2.0 ** 17 + 30) * U * size).all()


@pytest.mark.parametrize("cols", [200, 4096])
def test_what_a_call_returns_can_be_resized_and_saved_alone(fp8, cols):
    """Every result has memory of its own: growing one moves it, and leaves the others."""
    x, w = torch.randn(3, cols, device="cuda"), torch.randn(cols, device="cuda")
    n = fp8.rms_norm(x, w, residual=x, normed=True)
    for got in ([n.h, n.values, n.scales, n.y, n.rstd], [t for q in fp8.quantize(x, layout="both") for t in q],
                list(fp8.quantize(x, layout="tiles")), list(fp8.rms_norm_backward(x, n.h, w, n.rstd))):
        want = [bits_of(t).clone() for t in got]
        for i, t in enumerate(got):
            t.resize_(64, cols).view(torch.uint8).fill_(85)
            for j, u in enumerate(got):
                assert j <= i or torch.equal(bits_of(u), want[j]), (i, j)


@pytest.mark.parametrize("out", TYPES)
def test_autograd_sees_what_a_product_wrote(fp8, out):
    a, _ = operand(fp8, 1, 5, 300)
    b, _ = operand(fp8, 2, 7, 300)
    c = torch.zeros(5, 7, dtype=out, device="cuda")
    leaf = torch.ones(5, 7, dtype=out, device="cuda", requires_grad=True)
    product = leaf * c  # keeps c for its gradient
    before = c._version
    fp8.matmul(a, b, out=c)
    assert c._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.no_grad():  # as torch's own calls with out: only what would be recorded is refused
        assert torch.equal(fp8.matmul(a, b, out=leaf), c)
    with torch.inference_mode():
        held = torch.zeros(5, 7, dtype=out, device="cuda")
        assert torch.equal(fp8.matmul(a, b, out=held), c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_beyond_32_bits(fp8, dtype):
    """A y of 5e39 is an infinity, and its block NaN; the row's other blocks are what they are."""
    x, w = torch.zeros(2, 300, dtype=dtype), torch.full((300,), 3e38, dtype=dtype)
    x[0, 5], x[1, 200] = 1, -1
    for normed in (False, True):
        n = fp8.rms_norm(x.cuda(), w.cuda(), eps=0.0, normed=normed)
        s, q = bits(n.scales), host(n.values)
        assert s.tolist() == [[255, 127, 127], [127, 255, 127]]
        assert np.isnan(q[0, :128]).all() and np.isnan(q[1, 128:256]).all() and np.isnan(q).sum() == 256
        assert (q[~np.isnan(q)] == 0).all()
    y = host(n.y)
    assert y[0, 5] == np.inf and y[1, 200] == -np.inf and np.count_nonzero(y) == 2
