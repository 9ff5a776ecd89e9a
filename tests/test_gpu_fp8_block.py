"""8-bit products with block scales and their quantisers against 64-bit definitions."""
import pytest
import torch

from oracle import latent_oracle as L

pytestmark = pytest.mark.gpu

BF16, F32 = 2.0 ** -8, 2.0 ** -24
DEV = "cuda"


def _status():
    from transarch_b200 import _lib
    return _lib.read_status(torch.device(DEV))


def rows(m, k, g, f32=False):
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))
    return x if f32 else x.bfloat16()


@pytest.mark.parametrize("m,k,width,offset,f32,ue8m0", [
    (1, 16, 16, 0, False, False), (3, 7168, 7168, 0, False, True), (17, 144, 200, 8, False, True),
    (65, 1536, 1600, 3, False, False), (9, 272, 272, 0, True, True), (8, 128, 131, 2, True, False)])
def test_quantise_rows(m, k, width, offset, f32, ue8m0):
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(m + k)
    full = rows(m, width, g, f32)
    if m > 2:
        full[1] = 0
        full[2] *= 1e-20
    x = full[:, offset:offset + k]
    q, sc = K.fp8_quantise_rows(full.to(DEV)[:, offset:offset + k], scale_fmt="ue8m0" if ue8m0 else None)
    assert q.shape == (m, k) and sc.shape == (m, (k + 127) // 128)
    ref, ref_sc = L.quantise_groups(x, ue8m0)
    sc = sc.cpu().double()
    # one fp32 division; a power of two is exact
    assert bool(((sc - ref_sc).abs() <= (0 if ue8m0 else F32) * ref_sc).all())
    v = q.cpu().float().double() * sc.repeat_interleave(128, 1)[:, :k]
    step = sc.repeat_interleave(128, 1)[:, :k] * 2.0 ** -10
    assert bool(((v - x.double()).abs() <= 2.0 ** -4 * x.double().abs() * (1 + 1e-6) + step).all())
    if ue8m0:
        assert torch.equal(q.cpu().float().double(), ref)


@pytest.mark.parametrize("n,k,f32", [(128, 128, False), (200, 272, False), (576, 1536, True), (1, 16, True), (130, 400, False)])
@pytest.mark.parametrize("ue8m0", [False, True])
def test_quantise_blocks(n, k, f32, ue8m0):
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(n)
    w = rows(n, k + 16, g, f32)
    q, sc = K.fp8_quantise_blocks(w.to(DEV)[:, :k], scale_fmt="ue8m0" if ue8m0 else None)
    w = w[:, :k].double()
    sc, q = sc.cpu().double(), q.cpu().float().double()
    for r in range(0, n, 128):
        for c in range(0, k, 128):
            blk = w[r:r + 128, c:c + 128]
            top = blk.abs().max().clamp_min(1e-10) / 448
            s = sc[r // 128, c // 128]
            if ue8m0:
                assert float(torch.log2(s)) == round(float(torch.log2(s))) and s >= top * (1 - F32) and s < 2 * top
            else:
                assert abs(float(s - top)) <= F32 * float(top)
            v = q[r:r + 128, c:c + 128] * s
            assert bool(((v - blk).abs() <= 2.0 ** -4 * blk.abs() * (1 + 1e-6) + s * 2.0 ** -10).all())


def operands(m, n, k, g):
    a = (torch.randn(m, k, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    w = (torch.randn(n, k, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    G = (k + 127) // 128
    sa = torch.exp(torch.randn(m, G, generator=g)) / 300
    sw = torch.exp(torch.randn((n + 127) // 128, G, generator=g)) / 300
    return a, sa, w, sw


def check_product(a, sa, w, sw, y):
    ref, mass = L.block_matmul(a.float(), sa, w.float(), sw)
    G = sa.shape[1]
    # 128 products summed in the tensor pipe (each addition may cut a bit), G scaled additions in fp32
    bound = (128 * 2 * F32 + (G + 2) * F32) * mass + (BF16 if y.dtype == torch.bfloat16 else F32) * ref.abs()
    err = (y.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("m,n,k", [
    (1, 128, 7168), (1, 1, 16), (16, 200, 128), (17, 8192, 1536), (33, 129, 272), (64, 576, 7168), (100, 2112, 400),
    (128, 128, 128), (129, 256, 256), (300, 1000, 656), (333, 2112, 7168), (1025, 2600, 1040)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_product(m, n, k, out):
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(m + n + k)
    a, sa, w, sw = operands(m, n, k, g)
    y = K.fp8_block_matmul(a.to(DEV), sa.to(DEV), w.to(DEV), sw.to(DEV), out_dtype=out)
    assert _status() == 0 and y.dtype == out
    check_product(a, sa, w, sw, y)


def test_product_strides_and_untouched_columns():
    """Operands and result inside wider tensors, scales in either order; what lies beside the result stays."""
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(2)
    for m, n, k in ((5, 77, 144), (150, 333, 272)):
        a, sa, w, sw = operands(m, n, k, g)
        wide_a = torch.zeros(m, k + 48, dtype=torch.float8_e4m3fn, device=DEV)
        wide_a[:, 16:16 + k] = a.to(DEV)
        wide_w = torch.zeros(n, k + 32, dtype=torch.float8_e4m3fn, device=DEV)
        wide_w[:, 32:] = w.to(DEV)
        for odd in (0, 1):
            out = torch.full((m, n + 9), 3.0, dtype=torch.bfloat16, device=DEV)
            y = out[:, 4 + odd:4 + odd + n]
            K.fp8_block_matmul(wide_a[:, 16:16 + k], sa.to(DEV).t().contiguous().t(), wide_w[:, 32:],
                               sw.to(DEV).t().contiguous().t(), out=y)
            check_product(a, sa, w, sw, y)
            assert bool((out[:, :4 + odd] == 3).all()) and bool((out[:, 4 + odd + n:] == 3).all())
    assert _status() == 0


def test_product_keeps_tokens_apart():
    """NaN and infinite values of one token reach its own row of the result and no other."""
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(4)
    for m in (20, 300):
        a, sa, w, sw = operands(m, 256, 512, g)
        clean = K.fp8_block_matmul(a.to(DEV), sa.to(DEV), w.to(DEV), sw.to(DEV))
        a.view(torch.uint8)[7, 3] = 0x7f
        sa[9, 1] = float("inf")
        y = K.fp8_block_matmul(a.to(DEV), sa.to(DEV), w.to(DEV), sw.to(DEV))
        keep = [i for i in range(m) if i not in (7, 9)]
        assert torch.equal(y[keep], clean[keep]) and bool(torch.isnan(y[7]).all()) and not bool(torch.isfinite(y[9]).any())


@pytest.mark.parametrize("m", [1, 64, 200])
def test_linear_is_quantise_and_product(m):
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(m)
    x, wt = rows(m, 1536, g), torch.randn(300, 1536, generator=g) / 40
    w, ws = K.fp8_quantise_blocks(wt.to(DEV))
    for fmt in (None, "ue8m0"):
        a, sa = K.fp8_quantise_rows(x.to(DEV), scale_fmt=fmt)
        y = K.fp8_block_linear(x.to(DEV), w, ws, scale_fmt=fmt)
        assert torch.equal(y, K.fp8_block_matmul(a, sa, w, ws))
        check_product(a.cpu(), sa.cpu(), w.cpu(), ws.cpu(), y)
    again = K.fp8_block_linear(x.to(DEV), w, ws, scale_fmt="ue8m0")
    assert torch.equal(again, y)                               # split sums are added in a fixed order


def test_product_captured_and_on_another_stream():
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(6)
    x = rows(40, 2048, g).to(DEV)
    w, ws = K.fp8_quantise_blocks(torch.randn(500, 2048, generator=g).to(DEV))
    ref = K.fp8_block_linear(x, w, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = K.fp8_block_linear(x, w, ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, ref)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = K.fp8_block_linear(x, w, ws)
    for _ in range(2):
        x.copy_(rows(40, 2048, g))
        graph.replay()
        assert torch.equal(y, K.fp8_block_linear(x, w, ws))


@pytest.mark.parametrize("m,n,k", [(5, 20000, 144), (70, 20000, 144), (2049, 2600, 144), (129, 128, 7168), (400, 300, 2064)])
def test_product_more_tiles_than_multiprocessors_and_split_wide(m, n, k):
    """Persistent CTAs that take several tiles, in both kernels, and the wide kernel with K cut over a cluster."""
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(m + n + k)
    a, sa, w, sw = operands(m, n, k, g)
    dev = [t.to(DEV) for t in (a, sa, w, sw)]
    for dtype in (torch.bfloat16, torch.float32):
        check_product(a, sa, w, sw, K.fp8_block_matmul(*dev, out_dtype=dtype))
    assert _status() == 0


def test_division_is_correctly_rounded():
    """Codes of values over plain scales equal those of a true fp32 division, over many magnitudes."""
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(11)
    x = torch.randn(512, 1280, generator=g) * torch.exp2(torch.randint(-20, 20, (512, 1), generator=g).float())
    q, sc = K.fp8_quantise_rows(x.to(DEV))
    s = sc.cpu().repeat_interleave(128, 1)
    ref = (x / s).clamp(-448, 448).to(torch.float8_e4m3fn)                # CPU division: correctly rounded
    assert torch.equal(q.cpu().view(torch.uint8), ref.view(torch.uint8))
    assert torch.equal(sc.cpu(), x.view(512, 10, 128).abs().amax(2) / 448)


@pytest.mark.parametrize("m,over,k,out", [
    (5, 2, 2064, torch.bfloat16), (30, 7, 2064, torch.float32), (40, 2, 2064, torch.bfloat16), (128, 18, 2064, torch.bfloat16),
    (200, 1, 4112, torch.float32), (200, 17, 7184, torch.bfloat16)])
def test_product_whose_last_tiles_are_a_second_launch(m, over, k, out):
    """A few tiles more than whole waves of multiprocessors, eager, captured and with the activations quantised on the way."""
    from transarch_b200 import kernels as K
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n = (sms // 2 + over) * 256 - 40 if m > 128 else (sms + over) * 128 - 40
    g = torch.Generator().manual_seed(m + over)
    a, sa, w, sw = operands(m, n, k, g)
    d = [t.to(DEV) for t in (a, sa, w, sw)]
    y = K.fp8_block_matmul(*d, out_dtype=out)
    check_product(a, sa, w, sw, y)
    x = torch.randn(m, k, generator=g).bfloat16().to(DEV)
    lin = K.fp8_block_linear(x, d[2], d[3], out_dtype=out)
    assert torch.equal(lin, K.fp8_block_matmul(*K.fp8_quantise_rows(x), d[2], d[3], out_dtype=out))
    got, got_lin = torch.zeros_like(y), torch.zeros_like(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.fp8_block_matmul(*d, out=got)
        K.fp8_block_linear(x, d[2], d[3], out=got_lin)
    for _ in range(3):
        got.zero_()
        got_lin.zero_()
        graph.replay()
        assert torch.equal(got, y) and torch.equal(got_lin, lin)
    assert _status() == 0
