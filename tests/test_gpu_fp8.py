"""The 8-bit floating point product (e4m3, one scale per block of 128) through the C ABI against 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from antfly_amd import _lib, kernels  # noqa: E402
from antfly_amd._lib import Buffer  # noqa: E402
from tests import fp8_ref as F  # noqa: E402
from tests import gpu_util as G  # noqa: E402


def activations(rng, rows, in_dim):
    x = rng.standard_normal((rows, in_dim)).astype(np.float32)
    x[:, rng.random(in_dim) < 0.01] *= 30
    x[rng.random((rows, in_dim)) < 0.002] = 0
    return x


def guarded(rows, out_dim):
    """A result between two guards that nothing may write."""
    whole = torch.full((rows * out_dim + 128,), float("nan"), dtype=torch.float32, device=G.DEV)
    return whole, whole[64:64 + rows * out_dim].view(rows, out_dim)


def guards_hold(whole):
    return bool(torch.isnan(whole[:64]).all() and torch.isnan(whole[-64:]).all())


def product(x, w, w_scales, bias=None, residual=None, activation=0, quantized=False, lend=True):
    rows, in_dim = x.shape
    out_dim = w.shape[0]
    keep = [G.to_dev(w), G.to_dev(w_scales)]
    extra = {"activation": activation}
    for name, value in (("bias", bias), ("residual", residual)):
        if value is not None:
            keep.append(G.to_dev(value.astype(np.float32)))
            extra[name] = G.buf(keep[-1])
    whole, y = guarded(rows, out_dim)
    size = kernels.linearFp8WorkspaceBytes(rows, in_dim, out_dim)
    ws = torch.full((size + 256,), 0xFF, dtype=torch.uint8, device=G.DEV)
    extra["workspace"] = Buffer(ws.data_ptr(), size) if lend else kernels.NO_BUFFER
    if quantized:
        codes, scales = F.quantize(x)
        keep += [G.to_dev(codes), G.to_dev(scales)]
        kernels.launchMatmulFp8F32(G.stream(), G.buf(y), G.buf(keep[-2]), G.buf(keep[-1]), G.buf(keep[0]), G.buf(keep[1]), rows,
                                   in_dim, out_dim, **extra)
    else:
        keep.append(G.to_dev(x))
        kernels.launchLinearFp8F32(G.stream(), G.buf(y), G.buf(keep[-1]), G.buf(keep[0]), G.buf(keep[1]), rows, in_dim, out_dim,
                                   **extra)
    torch.cuda.synchronize()
    assert guards_hold(whole) and bool((ws[size:] == 0xFF).all())
    return y.cpu().numpy()


@pytest.mark.parametrize("rows,in_dim", [(1, 16), (1, 128), (3, 144), (7, 4096), (33, 2000), (130, 272)])
def test_quantizer_bit_exact(rows, in_dim):
    print(f"case: quantize_fp8 rows={rows} in={in_dim}", flush=True)
    rng = np.random.default_rng(rows + in_dim)
    x = activations(rng, rows, in_dim) * np.exp(rng.uniform(-20, 20, (rows, 1))).astype(np.float32)
    x[0, :16] = 0  # (in_dim 16: a block of zeros)
    if rows > 2:
        x[1] = 2.0 ** -130  # below what a scale is made from: codes of zero
        x[2, 3] = np.nan
    if rows > 6:
        x[3, 5] = np.inf
        x[4] = np.float32(2.0 ** 120) * np.sign(x[4] + 0.1)
        x[5, :8] = [448, 432, 416, 1.0625, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, -0.0]  # ties
    codes, scales = F.quantize(x)
    q = torch.full((rows * in_dim + 64,), 0xAA, dtype=torch.uint8, device=G.DEV)
    s = torch.full((scales.size + 16,), -1.0, dtype=torch.float32, device=G.DEV)
    xd = G.to_dev(x)
    kernels.launchQuantizeFp8(G.stream(), G.buf(q[:rows * in_dim]), G.buf(s[:scales.size]), G.buf(xd), rows, in_dim)
    torch.cuda.synchronize()
    got = q.cpu().numpy()
    assert (got[rows * in_dim:] == 0xAA).all() and (s[scales.size:] == -1.0).all()
    got = got[:rows * in_dim].reshape(rows, in_dim)
    bad = np.isnan(F.VALUES[codes])
    assert np.array_equal(np.isnan(F.VALUES[got]), bad)
    assert np.array_equal(got[~bad], codes[~bad])
    assert np.array_equal(s[:scales.size].cpu().numpy().view(np.uint32), scales.reshape(-1).view(np.uint32))


SHAPES = [(1, 16, 1), (1, 4096, 512), (2, 128, 130), (5, 4096, 1000), (16, 1040, 257), (17, 2000, 96), (33, 4112, 300), (48, 14336, 64),
          (64, 272, 1111), (65, 384, 129), (129, 144, 1000), (300, 1152, 777), (1, 14336, 2048), (8, 5632, 2048), (97, 4096, 640)]


@pytest.mark.parametrize("rows,in_dim,out_dim", SHAPES)
@pytest.mark.parametrize("quantized", [False, True])
def test_product(rows, in_dim, out_dim, quantized):
    print(f"case: fp8 product rows={rows} in={in_dim} out={out_dim} quantized={quantized}", flush=True)
    rng = np.random.default_rng(rows * 7 + in_dim + out_dim)
    x, (w, w_scales) = activations(rng, rows, in_dim), F.weights(rng, out_dim, in_dim)
    want, off = F.matmul(*F.quantize(x), w, w_scales)
    got = product(x, w, w_scales, quantized=quantized)
    assert (np.abs(got - want) <= off).all(), float((np.abs(got - want) / off).max())
    assert np.linalg.norm(got - want) <= 5e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("out_dim", [6001, 10239, 10241, 14336])
@pytest.mark.parametrize("rows,in_dim", [(1, 272), (3, 2000), (16, 144), (16, 2048), (17, 272), (32, 656)])
def test_product_many_columns(rows, in_dim, out_dim):
    """Both sides of where workgroups get smaller."""
    test_product(rows, in_dim, out_dim, rows % 2 == 0)


@pytest.mark.parametrize("rows,in_dim,out_dim", [(33, 2048, 4096), (48, 1040, 4097), (48, 4096, 6000), (41, 656, 10241), (96, 2064, 4111), (49, 2048, 4096)])
def test_product_up_to_three_sixteens_a_workgroup(rows, in_dim, out_dim):
    test_product(rows, in_dim, out_dim, rows % 2 == 0)


@pytest.mark.parametrize("rows,in_dim,out_dim", [(2048, 1024, 4000), (1100, 2192, 4096), (8193, 128, 1040)])
def test_product_many_rows(rows, in_dim, out_dim):
    """A prompt's sizes, with the activations' scales spread: every row of a sample against 64 bits."""
    print(f"case: fp8 product rows={rows} in={in_dim} out={out_dim}", flush=True)
    rng = np.random.default_rng(rows)
    x, (w, w_scales) = activations(rng, rows, in_dim), F.weights(rng, out_dim, in_dim)
    x *= np.exp(rng.uniform(-3, 3, (rows, 1))).astype(np.float32)
    got = product(x, w, w_scales)
    sample = np.unique(np.r_[0, 1, 63, 64, 127, 128, 255, 256, rows - 130, rows - 2, rows - 1, rng.integers(0, rows, 40)])
    want, off = F.matmul(*F.quantize(x[sample]), w, w_scales)
    assert (np.abs(got[sample] - want) <= off).all()
    assert np.isfinite(got).all()


@pytest.mark.parametrize("rows,in_dim,out_dim", [(512, 14336, 1024), (300, 8192, 2049), (128, 14336, 2000)])
def test_shares_of_k(rows, in_dim, out_dim):
    """A small grid on a long K: its blocks shared out over workgroups with a workspace lent, and not without one."""
    print(f"case: fp8 shares rows={rows} in={in_dim} out={out_dim}", flush=True)
    rng = np.random.default_rng(rows)
    x, (w, w_scales) = activations(rng, rows, in_dim), F.weights(rng, out_dim, in_dim)
    bias, residual = rng.standard_normal(out_dim).astype(np.float32), rng.standard_normal((rows, out_dim)).astype(np.float32)
    sample = np.unique(np.r_[0, 31, 64, 127, rows - 1, rng.integers(0, rows, 12)])
    y, off = F.matmul(*F.quantize(x[sample]), w, w_scales)
    want = np.where(y + bias < 0, 0.0, y + bias) + residual[sample]
    off = off + 2.0 ** -22 * (np.abs(y) + np.abs(want))
    assert kernels.linearFp8WorkspaceBytes(rows, in_dim, out_dim) > rows * in_dim + 2 * rows * out_dim * 4
    for quantized, lend in ((False, True), (True, True), (True, False)):
        got = product(x, w, w_scales, bias, residual, 1, quantized=quantized, lend=lend)
        assert (np.abs(got[sample] - want) <= off).all() and np.isfinite(got).all()


@pytest.mark.parametrize("rows,in_dim,out_dim", [(1, 512, 300), (5, 2000, 130), (40, 144, 257), (300, 640, 1111), (1100, 256, 4100)])
@pytest.mark.parametrize("activation", [0, 1, 2, 3])
def test_epilogue(rows, in_dim, out_dim, activation):
    """act(XW + b) + r: the activations' slopes are at most 1.13, their functions a few units in the last place, the sums two
    more roundings."""
    print(f"case: fp8 epilogue rows={rows} in={in_dim} out={out_dim} act={activation}", flush=True)
    rng = np.random.default_rng(rows + activation)
    x, (w, w_scales) = activations(rng, rows, in_dim), F.weights(rng, out_dim, in_dim)
    w_scales /= np.sqrt(in_dim) * 10
    bias, residual = rng.standard_normal(out_dim).astype(np.float32), rng.standard_normal((rows, out_dim)).astype(np.float32)
    y, off = F.matmul(*F.quantize(x), w, w_scales)
    inside = y + bias
    want = F.activate(inside, activation) + residual
    off = 1.2 * (off + 2.0 ** -23 * np.abs(inside)) + 2.0 ** -20 * (np.abs(F.activate(inside, activation)) + 1e-3) + 2.0 ** -23 * np.abs(want)
    got = product(x, w, w_scales, bias, residual, activation)
    assert (np.abs(got - want) <= off).all()
    got = product(x, w, w_scales, None, residual, activation, quantized=True, lend=False)
    want = F.activate(y, activation) + residual
    assert (np.abs(got - want) <= off + 1.2 * 2.0 ** -23 * np.abs(y)).all()


def test_residual_in_place_and_rows_that_are_no_numbers():
    rng = np.random.default_rng(5)
    rows, in_dim, out_dim = 20, 272, 96
    x, (w, w_scales) = activations(rng, rows, in_dim), F.weights(rng, out_dim, in_dim)
    x[3, 7], x[9, 200], x[11] = np.nan, np.inf, 0
    yd = G.to_dev(rng.standard_normal((rows, out_dim)).astype(np.float32))
    before = yd.cpu().numpy().astype(np.float64)
    xd, wd, sd = G.to_dev(x), G.to_dev(w), G.to_dev(w_scales)
    ws = torch.empty(kernels.linearFp8WorkspaceBytes(rows, in_dim, out_dim), dtype=torch.uint8, device=G.DEV)
    kernels.launchLinearFp8F32(G.stream(), G.buf(yd), G.buf(xd), G.buf(wd), G.buf(sd), rows, in_dim, out_dim, residual=G.buf(yd),
                               workspace=G.buf(ws))
    torch.cuda.synchronize()
    got = yd.cpu().numpy()
    bad = np.zeros(rows, bool)
    bad[[3, 9]] = True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()  # a bad row stays its own
    want, off = F.matmul(*F.quantize(x[~bad]), w, w_scales)
    want += before[~bad]
    assert (np.abs(got[~bad] - want) <= off + 2.0 ** -23 * np.abs(want)).all()
    assert np.array_equal(got[11], before[11].astype(np.float32))


@pytest.mark.parametrize("rows", [1, 6, 40, 200])
def test_other_stream_and_replayed_graph(rows):
    """The launches follow the stream that they are given, and a captured call gives the eager call's bits on every replay."""
    print(f"case: fp8 stream and graph rows={rows}", flush=True)
    rng = np.random.default_rng(rows)
    in_dim, out_dim = 1040, 520
    w, w_scales = F.weights(rng, out_dim, in_dim)
    wd, sd = G.to_dev(w), G.to_dev(w_scales)
    inputs = [activations(rng, rows, in_dim) for _ in range(3)]
    xd, y = G.to_dev(inputs[0]), torch.empty(rows, out_dim, dtype=torch.float32, device=G.DEV)
    ws = torch.empty(kernels.linearFp8WorkspaceBytes(rows, in_dim, out_dim), dtype=torch.uint8, device=G.DEV)

    def call():
        kernels.launchLinearFp8F32(G.stream(), G.buf(y), G.buf(xd), G.buf(wd), G.buf(sd), rows, in_dim, out_dim, workspace=G.buf(ws))

    eager = [product(x, w, w_scales) for x in inputs]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        xd.copy_(torch.from_numpy(inputs[1]))
        call()
        copied = y.clone()
    side.synchronize()
    assert np.array_equal(copied.cpu().numpy(), eager[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in (0, 1, 2, 0):
        xd.copy_(torch.from_numpy(inputs[i]))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(y.cpu().numpy(), eager[i])


@pytest.mark.parametrize("most,fewer,in_dim,out_dim", [(258, (257, 200, 40, 3), 4096, 4096), (85, (84, 65), 8192, 4096)])
def test_a_workspace_of_more_rows_does_for_fewer(most, fewer, in_dim, out_dim):
    """The shares' sums of fewer rows may take more room than all that more rows ask for: then there are fewer shares."""
    size = kernels.linearFp8WorkspaceBytes(most, in_dim, out_dim)
    assert any(kernels.linearFp8WorkspaceBytes(rows, in_dim, out_dim) > size for rows in fewer)
    rng = np.random.default_rng(most)
    w, w_scales = F.weights(rng, out_dim, in_dim)
    wd, sd = G.to_dev(w), G.to_dev(w_scales)
    ws = torch.full((size + 256,), 0xFF, dtype=torch.uint8, device=G.DEV)
    for rows in fewer:
        print(f"case: fp8 workspace of {most} rows, {rows} rows in={in_dim} out={out_dim}", flush=True)
        x = activations(rng, rows, in_dim)
        whole, y = guarded(rows, out_dim)
        xd = G.to_dev(x)
        kernels.launchLinearFp8F32(G.stream(), G.buf(y), G.buf(xd), G.buf(wd), G.buf(sd), rows, in_dim, out_dim, workspace=G.buf(ws[:size]))
        torch.cuda.synchronize()
        assert guards_hold(whole) and bool((ws[size:] == 0xFF).all())
        sample = np.unique(np.r_[0, rows - 1, rng.integers(0, rows, 10)])
        want, off = F.matmul(*F.quantize(x[sample]), w, w_scales)
        got = y.cpu().numpy()
        assert (np.abs(got[sample] - want) <= off).all() and np.isfinite(got).all()
