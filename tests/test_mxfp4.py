"""Microscaled fp4: quantisation, its inverse and the product, against their definitions in 64 bits.

Tolerances, derived beforehand:
  * codes, scales and dequantised values are whole numbers or exact: they are equal.
  * a product of two e2m1 values times scales of 2^-1, 1 and 2 is a multiple of 2^-4 and at most 144; K of them
    stay a multiple of 2^-4 below 144 K, so for K <= 7281 every partial sum is below 2^24 * 2^-4 and exact in
    fp32 in any order: the fp32 output is equal, the bf16 output is that rounded once.
  * with scales over a wide range each of K additions may be off by 2^-23 of the sum of magnitudes (a truncated
    addition; a rounded one is half of it).
"""
import pytest

torch = pytest.importorskip("torch")

from kubernetes_amd.ops import hip_kernels as hk  # noqa: E402

TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    hk.load()   # must load: no fallback
    return torch.device("cuda")


# ---------------------------------------------------------------------------
# the definitions, on the CPU in 64 bits

def values_of(q, scale):
    q, scale = q.cpu(), scale.cpu()
    c = torch.stack((q & 15, q >> 4), dim=-1).reshape(*q.shape[:-1], -1)
    e, f, neg = (c >> 1 & 3).double(), (c & 1).double(), c >= 8
    v = torch.where(e == 0, 0.5 * f, (1 + 0.5 * f) * torch.exp2(e - 1))
    v = torch.where(neg, -v, v)
    s = torch.exp2(scale.double() - 127)
    s[scale == 255] = float("nan")
    return v * s.repeat_interleave(32, dim=-1)


def quantized(x):
    """Codes and scales of x [rows, K] by the definition."""
    x = x.cpu().double()
    rows, K = x.shape
    nb = -(-K // 32)
    v = torch.zeros(rows, nb * 32, dtype=torch.float64)
    v[:, :K] = x
    v = v.view(rows, nb, 32)
    bad = ~torch.isfinite(v).all(dim=2)
    v = torch.where(bad[:, :, None], 0.0, v)
    amax = v.abs().amax(dim=2)
    _, e = torch.frexp(amax)
    s = torch.where(amax > 0, (e - 1 - 2 + 127).clamp(min=0), 0)
    w = v / torch.exp2(s.double() - 127)[:, :, None]
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    d = (w.abs().clamp(max=6)[..., None] - grid).abs()
    near = d == d.amin(dim=-1, keepdim=True)
    code = torch.arange(8).expand_as(near)
    # of two equally near codes the even one
    code = torch.where(near, torch.where(code % 2 == 0, code, code + 8), 99).amin(dim=-1) % 8
    code = (code + torch.where(torch.signbit(w), 8, 0)).to(torch.uint8)
    code[bad] = 0
    s[bad] = 255
    code = code.view(rows, nb * 32)
    return code[:, 0::2] | (code[:, 1::2] << 4), s.to(torch.uint8)


def operand(rows, nb, seed, scales=(126, 127, 128), device="cuda"):
    """Random codes and scales of the given range."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (rows, 16 * nb), generator=g, dtype=torch.uint8)
    s = torch.tensor(scales, dtype=torch.uint8)[torch.randint(0, len(scales), (rows, nb), generator=g)]
    return q.to(device), s.to(device)


def test_definition_against_itself():
    """Quantising what codes stand for gives it back, and the error is at most half a step."""
    x = torch.randn(7, 100) * torch.logspace(-30, 30, 7)[:, None]
    q, s = quantized(x)
    v = values_of(q, s)
    q2, s2 = quantized(v)
    assert torch.equal(values_of(q2, s2), v)
    amax = torch.nn.functional.pad(x.double(), (0, 28)).view(7, 4, 32).abs().amax(dim=2, keepdim=True)
    # steps are 2^(e - 2) of the block's 2^e at most; above 6/4 2^e values saturate
    err = (v.view(7, 4, 32) - torch.nn.functional.pad(x.double(), (0, 28)).view(7, 4, 32)).abs()
    assert (err <= amax / 4).all()


# ---------------------------------------------------------------------------
# refusals: before anything is launched, so on the CPU

def test_refusals():
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
        hk.mxfp4_quantize(torch.zeros(4, 32, dtype=torch.float64))
    with pytest.raises(ValueError, match="dimension"):
        hk.mxfp4_quantize(torch.zeros(()))
    with pytest.raises(ValueError, match="GPU"):
        hk.mxfp4_quantize(torch.zeros(4, 32))
    with pytest.raises(ValueError, match="uint8"):
        hk.mxfp4_dequantize(q.int(), s)
    with pytest.raises(ValueError, match="uint8"):
        hk.mxfp4_dequantize(q, s.float())
    with pytest.raises(ValueError, match="16 \\* blocks"):
        hk.mxfp4_dequantize(q, s[:, :1])
    with pytest.raises(ValueError, match="16 \\* blocks"):
        hk.mxfp4_dequantize(q, s[:3])
    with pytest.raises(ValueError, match="16 \\* blocks"):
        hk.mxfp4_dequantize(q[0], s)
    for k in (-1, 0, 32, 65):
        with pytest.raises(ValueError, match="k="):
            hk.mxfp4_dequantize(q, s, k=k)
    with pytest.raises(ValueError, match="gives"):
        hk.mxfp4_dequantize(q, s, dtype=torch.float64)
    with pytest.raises(ValueError, match="GPU"):
        hk.mxfp4_dequantize(q, s, k=33)
    with pytest.raises(ValueError, match="gemm_mxfp4_nt needs codes"):
        hk.gemm_mxfp4_nt(q, s, q[:, :16], s[:, :1])
    with pytest.raises(ValueError, match="gemm_mxfp4_nt needs codes"):
        hk.gemm_mxfp4_nt(q[None], s[None], q[None], s[None])
    with pytest.raises(ValueError, match="gemm_mxfp4_nt b"):
        hk.gemm_mxfp4_nt(q, s, q, s[:2])
    with pytest.raises(ValueError, match="GPU"):
        hk.gemm_mxfp4_nt(q, s, q, s)


# ---------------------------------------------------------------------------
# quantisation

def check_quantize(x):
    q, s = hk.mxfp4_quantize(x)
    K = x.shape[-1]
    want_q, want_s = quantized(x.reshape(-1, K))
    assert q.shape == (*x.shape[:-1], 16 * -(-K // 32)) and s.shape == (*x.shape[:-1], -(-K // 32))
    assert torch.equal(s.cpu().reshape(want_s.shape), want_s)
    assert torch.equal(q.cpu().reshape(want_q.shape), want_q)
    return q, s


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K", [(1, 32), (1, 1), (3, 31), (5, 33), (2, 64), (17, 100), (1, 8192), (64, 256),
                                    (33, 1025), (300, 7), (129, 520), (257, 96), (1000, 264)])
def test_quantize(gpu, dtype, rows, K):
    g = torch.Generator().manual_seed(rows * K)
    x = (torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-12, 9, (rows, 1), generator=g).float())).to(dtype)
    check_quantize(x.to(gpu))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_every_value(gpu, dtype):
    """Every 16-bit pattern (for fp32: every such upper half), each beside a block maximum that puts it on
    another part of the grid, subnormals and the largest values among them."""
    bits = torch.arange(65536, dtype=torch.int32)
    if dtype == torch.float32:
        v = (bits * 65536 + (bits * 40503) % 65536).view(torch.float32)
    else:
        v = bits.to(torch.int16).view(dtype)
    v = v[torch.isfinite(v)]
    for shift in (0, 1, 2, 5):
        x = torch.zeros(v.numel(), 32, dtype=dtype)
        x[:, 3] = v
        x[:, 17] = (v.double() * 2.0 ** shift).clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype)
        x[:, 30] = -(v.double() * 0.75).to(dtype)
        check_quantize(x.to(gpu))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_ties_zeros_and_blocks_without_an_answer(gpu, dtype):
    t = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.0, 7.5, 0.2499, 0.26, -0.0, -0.25, -5.0, 4.0])
    x = torch.zeros(8, 96)
    x[0, 16:32] = t
    x[1, :16] = t * 2.0 ** -14
    x[2, 40] = float("nan")
    x[3, 0] = float("inf")
    x[4, 95] = -float("inf")
    x[5, 64] = -0.0
    x[6] = torch.finfo(dtype).max
    x[7] = torch.finfo(dtype).tiny
    q, s = check_quantize(x.to(dtype).to(gpu))
    assert s[2, 1] == 255 and s[3, 0] == 255 and s[4, 2] == 255 and s[5].sum() == 0
    v = hk.mxfp4_dequantize(q, s, dtype=torch.float32)
    assert torch.isnan(v[2, 32:64]).all() and torch.isfinite(v[2, :32]).all() and torch.isfinite(v[2, 64:]).all()
    assert torch.isfinite(v[6]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K", [(1, 64), (2, 1), (31, 33), (64, 32), (65, 100), (128, 256), (130, 259), (257, 513), (8, 4097),
                                    (127, 287), (640, 1000)])
def test_quantize_strides(gpu, dtype, rows, K):
    g = torch.Generator().manual_seed(K)
    x = torch.randn(K, rows, generator=g).to(dtype).to(gpu)
    check_quantize(x.t())                                    # blocks along the other axis
    wide = torch.randn(K, rows + 13, generator=g).to(dtype).to(gpu)
    check_quantize(wide[:, 5:5 + rows].t())
    check_quantize(torch.randn(1, rows, generator=g).to(dtype).to(gpu).expand(K, rows).t())
    bad = x.clone()
    bad[K // 2, rows // 2], bad[K - 1, 0] = float("nan"), -float("inf")
    check_quantize(bad.t())
    check_quantize(torch.randn(rows, K + 9, generator=g).to(dtype).to(gpu)[:, 3:3 + K])   # unaligned rows
    check_quantize(torch.randn(rows, 2 * K, generator=g).to(dtype).to(gpu)[:, ::2])
    check_quantize(torch.randn(1, K, generator=g).to(dtype).to(gpu).expand(rows, K))
    check_quantize(torch.randn(rows, 1, generator=g).to(dtype).to(gpu).expand(rows, K))
    check_quantize(torch.randn(3 * rows, K, generator=g).to(dtype).to(gpu)[::3])


@pytest.mark.gpu
def test_quantize_overlapping_and_negated_views(gpu):
    g = torch.Generator().manual_seed(31)
    row = torch.randn(4 * 96, generator=g).to(gpu)
    imag = torch.view_as_complex(row.view(4, 48, 2)).conj().imag
    for x in (row[:96].expand(7, 96), row[:70, None].expand(70, 40), row.unfold(0, 96, 1), row.unfold(0, 96, 5), imag,
              imag.t(), imag[:, 5:6]):
        check_quantize(x)


@pytest.mark.gpu
def test_quantize_shapes(gpu):
    x = torch.randn(2, 3, 5, 70, device=gpu)
    check_quantize(x)
    check_quantize(x.transpose(0, 2))
    check_quantize(x.transpose(1, 3))
    check_quantize(torch.randn(77, device=gpu))
    for shape in ((0, 64), (4, 0), (0,), (3, 0, 8), (0, 33)):
        q, s = hk.mxfp4_quantize(torch.zeros(shape, device=gpu))
        nb = -(-shape[-1] // 32)
        assert q.shape == (*shape[:-1], 16 * nb) and s.shape == (*shape[:-1], nb)
        assert hk.mxfp4_dequantize(q, s, k=shape[-1]).shape == shape


# ---------------------------------------------------------------------------
# dequantisation

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_dequantize_every_code_and_scale(gpu, dtype):
    """All codes under all scales: 64-bit values rounded once to the type (infinity and subnormals included)."""
    q = (torch.arange(16, dtype=torch.uint8) * 17).expand(256, 16).contiguous()
    s = torch.arange(256, dtype=torch.uint8)[:, None]
    want = values_of(q, s).to(dtype)
    got = hk.mxfp4_dequantize(q.to(gpu), s.to(gpu), dtype=dtype).cpu()
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (3, 31), (5, 33), (17, 100), (300, 7), (129, 520), (2, 8191), (1000, 264)])
def test_dequantize(gpu, dtype, rows, k):
    q, s = operand(rows, -(-k // 32), k, scales=tuple(range(110, 140)))
    want = values_of(q, s)[:, :k].to(dtype)
    assert torch.equal(hk.mxfp4_dequantize(q, s, k=k, dtype=dtype).cpu(), want)
    if k % 32 == 0:
        assert torch.equal(hk.mxfp4_dequantize(q, s).cpu(), want.to(torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_round_trip_keeps_what_is_on_the_grid(gpu, dtype):
    x = torch.randn(64, 777, device=gpu).to(dtype)
    v = hk.mxfp4_dequantize(*hk.mxfp4_quantize(x), k=777, dtype=dtype)
    assert torch.equal(hk.mxfp4_dequantize(*hk.mxfp4_quantize(v), k=777, dtype=dtype), v)
    assert torch.equal(v.cpu(), values_of(*quantized(x))[:, :777].to(dtype))


# ---------------------------------------------------------------------------
# product

def product(a, sa, b, sb):
    return values_of(a, sa) @ values_of(b, sb).t()


SIZES = [(1, 1, 1), (1, 16, 4), (1, 4096, 8), (2, 17, 3), (7, 33, 5), (16, 16, 7), (16, 256, 128), (17, 48, 9), (31, 130, 12),
         (32, 512, 16), (33, 17, 1), (48, 64, 33), (64, 64, 8), (64, 1000, 17), (65, 129, 24), (100, 200, 31), (127, 128, 16),
         (128, 128, 64), (129, 127, 32), (200, 300, 40), (255, 257, 20), (256, 256, 8), (256, 512, 16), (257, 256, 24),
         (512, 768, 32), (520, 1000, 9), (700, 300, 65), (1024, 1024, 10), (2049, 130, 6), (130, 2049, 11)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,nb", SIZES)
def test_gemm(gpu, M, N, nb):
    a, sa = operand(M, nb, 1)
    b, sb = operand(N, nb, 2)
    want = product(a, sa, b, sb)
    assert torch.equal(hk.gemm_mxfp4_nt(a, sa, b, sb).cpu(), want.float())
    assert torch.equal(hk.gemm_mxfp4_nt(a, sa, b, sb, out_fp32=False).cpu(), want.float().to(torch.bfloat16))
    assert torch.equal(hk.gemm_mxfp4_nt(a, sa, b, sb, alpha=-0.25).cpu(), -0.25 * want.float())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(4096, 4096, 4096), (2048, 1024, 4096), (8192, 512, 1024), (1, 8192, 7264), (32, 4096, 4096),
                                   (300, 4096, 2048), (1000, 520, 264), (3000, 3001, 1111), (4097, 4095, 289),
                                   (4352, 4100, 1000), (8191, 2100, 600), (2100, 8200, 512), (4096, 4096, 256), (4096, 4096, 768)])
def test_gemm_large(gpu, M, N, K):
    """Exact as above; the oracle is a product in 64 bits on the GPU, whose sums of these are exact too."""
    a, sa = operand(M, -(-K // 32), 3)
    b, sb = operand(N, -(-K // 32), 4)
    want = values_of(a, sa).to(gpu) @ values_of(b, sb).to(gpu).t()
    assert torch.equal(hk.gemm_mxfp4_nt(a, sa, b, sb), want.float())
    assert torch.equal(hk.gemm_mxfp4_nt(a, sa, b, sb, out_fp32=False), want.float().to(torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("nb", [1, 2, 5, 7])
@pytest.mark.parametrize("M,N", [(64, 64), (97, 130), (2048, 2050), (2304, 1290), (4100, 4111)])
def test_gemm_short_k(gpu, M, N, nb):
    """Rows of fewer blocks than a tile has, in tiles of each size."""
    a, sa = operand(M, nb, 24)
    b, sb = operand(N, nb, 25)
    sa[M - 1, nb - 1] = sb[N // 2, 0] = 255
    want = (values_of(a, sa).to(gpu) @ values_of(b, sb).to(gpu).t()).float()
    for fp32, dtype in ((True, torch.float32), (False, torch.bfloat16)):
        torch.testing.assert_close(hk.gemm_mxfp4_nt(a, sa, b, sb, out_fp32=fp32), want.to(dtype), rtol=0, atol=0, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,nb", [(1, 33, 40), (40, 70, 9), (128, 300, 32), (300, 520, 40), (512, 512, 64)])
def test_gemm_wide_scales(gpu, M, N, nb):
    a, sa = operand(M, nb, 5, scales=tuple(range(100, 150)))
    b, sb = operand(N, nb, 6, scales=tuple(range(100, 150)))
    va, vb = values_of(a, sa), values_of(b, sb)
    got = hk.gemm_mxfp4_nt(a, sa, b, sb).cpu().double()
    bound = 32 * nb * 2.0 ** -23 * (va.abs() @ vb.abs().t())
    assert ((got - va @ vb.t()).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(16, 48), (200, 130), (512, 512)])
def test_gemm_scale_range_and_nan(gpu, M, N):
    """2^100 times 2^-100 is 1; too large is infinity; NaN reaches its row and column and no other."""
    nb = 12
    a, sa = operand(M, nb, 7)
    b, sb = operand(N, nb, 8)
    far = hk.gemm_mxfp4_nt(a, sa + 100, b, sb - 100)
    assert torch.equal(far, hk.gemm_mxfp4_nt(a, sa, b, sb))
    one = torch.full((M, 16 * nb), 0x22, dtype=torch.uint8, device=gpu), torch.full((M, nb), 254, dtype=torch.uint8, device=gpu)
    two = torch.full((N, 16 * nb), 0x22, dtype=torch.uint8, device=gpu), torch.full((N, nb), 254, dtype=torch.uint8, device=gpu)
    assert torch.isposinf(hk.gemm_mxfp4_nt(*one, *two)).all()
    want = product(a, sa, b, sb).float()
    sa, sb = sa.clone(), sb.clone()
    a[3], b[5] = 0, 0
    sa[3, nb - 1] = 255
    sb[5, 0] = 255
    got = hk.gemm_mxfp4_nt(a, sa, b, sb).cpu()
    nan = torch.zeros(M, N, dtype=torch.bool)
    nan[3], nan[:, 5] = True, True
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], want[~nan])


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,nb", [(3000, 3001, 12), (2600, 2500, 9), (4100, 300, 15)])
def test_gemm_nan_in_large_tiles(gpu, M, N, nb):
    """A NaN scale in the first block, in the last of a short tile of K, and in rows that two tiles cover."""
    a, sa = operand(M, nb, 20)
    b, sb = operand(N, nb, 21)
    want = hk.gemm_mxfp4_nt(a, sa, b, sb)
    for i in (0, 130, M - 200, M - 1):
        sa[i, nb - 1 if i % 2 else 0] = 255
        want[i] = float("nan")
    for j in (7, N - 1):
        sb[j, nb - 1] = 255
        want[:, j] = float("nan")
    torch.testing.assert_close(hk.gemm_mxfp4_nt(a, sa, b, sb), want, rtol=0, atol=0, equal_nan=True)


LONG = [(1, 1, 2048), (1, 500, 2041), (16, 100, 2059), (32, 64, 4100), (100, 7, 2304), (40, 70, 515), (300, 48, 519), (64, 64, 505),
        (64, 64, 1025), (100, 200, 777), (512, 500, 1024)]


def long_operand(rows, nb, seed):
    """Values up to 1.5: sums of some hundred thousand products in steps of 1/4 stay exact in 32 bits."""
    q, s = operand(rows, nb, seed, scales=(127,))
    return q & 0xBB, s


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,nb", LONG)
def test_gemm_long_k(gpu, M, N, nb):
    """A K that few workgroups would have for themselves is taken in parts. NaN of one part stays."""
    assert hk.load().kamd_gemm_mxfp4_nt_workspace(M, N, nb) >= 2 * M * N * 4
    a, sa = long_operand(M, nb, 26)
    b, sb = long_operand(N, nb, 27)
    want = (values_of(a, sa).to(gpu) @ values_of(b, sb).to(gpu).t()).float()
    for _ in range(2):
        assert torch.equal(hk.gemm_mxfp4_nt(a, sa, b, sb), want)
    assert torch.equal(hk.gemm_mxfp4_nt(a, sa, b, sb, out_fp32=False), want.to(torch.bfloat16))
    assert torch.equal(hk.gemm_mxfp4_nt(a, sa, b, sb, alpha=-0.25), -0.25 * want)
    sa[M - 1, nb - 1] = sb[0, 3] = 255
    want[M - 1] = want[:, 0] = float("nan")
    torch.testing.assert_close(hk.gemm_mxfp4_nt(a, sa, b, sb), want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.gpu
def test_gemm_long_k_twice_at_once(gpu):
    """Two products in parts on two streams, and in a graph that is replayed beside them: each has its own sums."""
    a, sa = long_operand(100, 777, 28)
    b, sb = long_operand(200, 777, 29)
    c, sc = long_operand(60, 777, 30)
    first, second = hk.gemm_mxfp4_nt(a, sa, b, sb), hk.gemm_mxfp4_nt(c, sc, b, sb)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = hk.gemm_mxfp4_nt(a, sa, b, sb)
    other = torch.cuda.Stream()
    for _ in range(3):
        held.zero_()
        graph.replay()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            y = [hk.gemm_mxfp4_nt(c, sc, b, sb) for _ in range(5)]
        x = [hk.gemm_mxfp4_nt(a, sa, b, sb) for _ in range(5)]
        torch.cuda.synchronize()
        assert torch.equal(held, first) and all(torch.equal(v, first) for v in x) and all(torch.equal(v, second) for v in y)


@pytest.mark.gpu
def test_gemm_same_rows_in_any_company(gpu):
    """A row's outputs are the same values whatever kernel its company has it computed by, where sums are exact."""
    b, sb = operand(4096, 20, 22)
    a, sa = operand(4096, 20, 23)
    want = hk.gemm_mxfp4_nt(a, sa, b, sb)
    for m in (1, 16, 17, 40, 64, 100, 256, 700, 2048):
        assert torch.equal(hk.gemm_mxfp4_nt(a[:m], sa[:m], b, sb), want[:m])
        assert torch.equal(hk.gemm_mxfp4_nt(b, sb, a[:m], sa[:m]).t(), want[:m])


@pytest.mark.gpu
def test_gemm_empty(gpu):
    for M, N, nb in ((0, 4, 2), (4, 0, 2), (0, 0, 0)):
        a, sa = operand(M, nb, 1)
        b, sb = operand(N, nb, 1)
        assert hk.gemm_mxfp4_nt(a, sa, b, sb).shape == (M, N)
    a, sa = operand(300, 0, 1)
    for fp32 in (True, False):
        torch.full((300, 300), 7.0, device=gpu)    # leave something behind in the allocator
        out = hk.gemm_mxfp4_nt(a, sa, a, sa, out_fp32=fp32)
        assert out.shape == (300, 300) and not out.any()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 150, 520])
def test_gemm_operands_as_they_come(gpu, M):
    """Column slices, steps, unaligned starts, torch's own 4-bit and scale types: the same result."""
    a, sa = operand(M, 12, 9)
    b, sb = operand(260, 12, 10)
    want = hk.gemm_mxfp4_nt(a, sa, b, sb)
    f4, e8 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
    assert torch.equal(hk.gemm_mxfp4_nt(a.view(f4), sa.view(e8), b.view(f4), sb.view(e8)), want)
    wide, wide_s = operand(M, 20, 11)
    wide[:, 64:256], wide_s[:, 4:16] = a, sa
    assert torch.equal(hk.gemm_mxfp4_nt(wide[:, 64:256], wide_s[:, 4:16], b, sb), want)
    flat = torch.zeros(a.numel() + 5, dtype=torch.uint8, device=gpu)
    flat[5:] = a.flatten()
    sflat = torch.zeros(sb.numel() + 3, dtype=torch.uint8, device=gpu)
    sflat[3:] = sb.flatten()
    assert torch.equal(hk.gemm_mxfp4_nt(flat[5:].view(a.shape), sa, b, sflat[3:].view(sb.shape)), want)
    assert torch.equal(hk.mxfp4_dequantize(flat[5:].view(a.shape), sa), hk.mxfp4_dequantize(a, sa))
    twice = a.repeat_interleave(2, 0)
    assert torch.equal(hk.gemm_mxfp4_nt(twice[::2], sa, b, sb), want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,nb", [(3, 50, 9), (70, 33, 17), (300, 400, 13), (513, 300, 20), (2100, 2050, 9),
                                    (4100, 4111, 13), (70, 65, 3), (2100, 2050, 5), (4100, 4111, 7)])
def test_gemm_writes_its_output_and_nothing_else(gpu, M, N, nb):
    """Launched into the middle of a larger buffer, the bytes before and behind stay."""
    a, sa = operand(M, nb, 12)
    b, sb = operand(N, nb, 13)
    for fp32, dtype in ((1, torch.float32), (0, torch.bfloat16)):
        buf = torch.full((M * N + 512,), 3.0, device=gpu, dtype=dtype)
        out = buf[256:256 + M * N]
        need = hk.load().kamd_gemm_mxfp4_nt_workspace(M, N, nb)
        ws = torch.full((need + 512,), 77, device=gpu, dtype=torch.uint8)
        rc = hk.load().kamd_gemm_mxfp4_nt_launch(a.data_ptr(), sa.data_ptr(), b.data_ptr(), sb.data_ptr(), out.data_ptr(),
                                                 M, N, nb, 1.0, fp32, ws.data_ptr() + 256, need, hk._stream(a))
        assert rc == 0
        assert (ws[:256] == 77).all() and (ws[256 + need:] == 77).all()
        assert (buf[:256] == 3).all() and (buf[256 + M * N:] == 3).all()
        assert torch.equal(out.view(M, N).cpu(), product(a, sa, b, sb).float().to(dtype))


# ---------------------------------------------------------------------------
# together

@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 5, 64, 333])
def test_a_layer_and_its_gradients(gpu, tokens):
    """Forward and both gradient products of y = x w^T, every product on operands that are quantised along the
    axis that it sums over: w's and dy's other axis from transposed views."""
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, 200, generator=g).to(torch.bfloat16).to(gpu)
    w = (torch.randn(264, 200, generator=g) * 0.05).to(torch.bfloat16).to(gpu)
    dy = torch.randn(tokens, 264, generator=g).to(torch.bfloat16).to(gpu)

    def close(got, left, right):
        va, vb = values_of(*quantized(left)), values_of(*quantized(right))
        bound = va.shape[1] * 2.0 ** -23 * (va.abs() @ vb.abs().t())
        assert ((got.cpu().double() - va @ vb.t()).abs() <= bound).all()

    close(hk.gemm_mxfp4_nt(*hk.mxfp4_quantize(x), *hk.mxfp4_quantize(w)), x, w)
    close(hk.gemm_mxfp4_nt(*hk.mxfp4_quantize(dy), *hk.mxfp4_quantize(w.t())), dy, w.t())
    close(hk.gemm_mxfp4_nt(*hk.mxfp4_quantize(dy.t()), *hk.mxfp4_quantize(x.t())), dy.t(), x.t())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_captured_and_replayed(gpu, tokens):
    """Two graphs of quantise, multiply, dequantise; replayed in turn on new inputs with eager calls between."""
    w = hk.mxfp4_quantize(torch.randn(520, 264, device=gpu))
    xs = [torch.randn(tokens, 264, device=gpu).to(torch.bfloat16) for _ in range(2)]

    def step(x):
        q, s = hk.mxfp4_quantize(x)
        return hk.gemm_mxfp4_nt(q, s, *w, out_fp32=False), hk.mxfp4_dequantize(q, s, k=264), hk.mxfp4_quantize(x.t())[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in xs:
            step(x)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(x))
        graphs.append(graph)
    for i in range(4):
        for x in xs:
            x.copy_(torch.randn(tokens, 264, device=gpu))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for x, out in zip(xs, outs):
            for got, want in zip(out, step(x)):
                assert torch.equal(got, want)


@pytest.mark.gpu
def test_on_another_stream(gpu):
    a, sa = operand(300, 40, 14)
    b, sb = operand(500, 40, 15)
    want = hk.gemm_mxfp4_nt(a, sa, b, sb)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            for _ in range(3):
                outs.append(hk.gemm_mxfp4_nt(a, sa, b, sb))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ---------------------------------------------------------------------------
# sizes whose offsets pass 32 bits

@pytest.mark.gpu
def test_quantize_behind_32_bits(gpu):
    """2^34 values and some rows: input offsets, output offsets and the count of lanes all pass 32 bits."""
    rows, K = (1 << 19) + 3, 32768
    x = torch.zeros(rows, K, device=gpu, dtype=torch.bfloat16)
    at = [0, 1, 65535, 65537, 1 << 18, (1 << 19) - 1, 1 << 19, rows - 1]
    x[at] = torch.randn(len(at), K, device=gpu).to(torch.bfloat16)
    q, s = hk.mxfp4_quantize(x)
    want_q, want_s = quantized(x[at])
    assert torch.equal(q[at].cpu(), want_q) and torch.equal(s[at].cpu(), want_s)
    assert q.count_nonzero() == q[at].count_nonzero() and s.count_nonzero() == s[at].count_nonzero()
    x.fill_(1.0)
    y = hk.mxfp4_dequantize(q, s)
    del x
    assert torch.equal(y[at].cpu().double(), values_of(want_q, want_s))
    assert y.count_nonzero() == y[at].count_nonzero()


@pytest.mark.gpu
def test_gemm_behind_32_bits(gpu):
    """An operand of more than 4 GiB, then an output of more than 2^31 values."""
    M, nb = 70001, 4096
    a = torch.zeros(M, 16 * nb, device=gpu, dtype=torch.uint8)
    sa = torch.full((M, nb), 127, device=gpu, dtype=torch.uint8)
    at = [0, 65535, 65536, M - 1]
    pick, _ = operand(len(at), nb, 16)
    pick &= 0x33     # values up to 1.5: 131072 products of at most 9 in steps of 1/4 stay exact
    a[at] = pick
    b, sb = operand(20, nb, 17, scales=(127,))
    got = hk.gemm_mxfp4_nt(a, sa, b, sb)
    assert torch.equal(got[at].cpu(), product(pick, sa[at], b, sb).float())
    assert got.count_nonzero() == got[at].count_nonzero()
    got_t = hk.gemm_mxfp4_nt(b, sb, a, sa)
    assert torch.equal(got_t, got.t())
    del a, sa, got, got_t
    a, sa = operand(46400, 1, 18)
    b, sb = operand(46401, 1, 19)
    got = hk.gemm_mxfp4_nt(a, sa, b, sb, out_fp32=False)
    for rows in (slice(0, 3), slice(23000, 23003), slice(46397, 46400)):
        assert torch.equal(got[rows].cpu(), product(a[rows], sa[rows], b, sb).float().to(torch.bfloat16))


def test_c_entries_refuse_bad_sizes():
    """The C entries check for themselves; nothing is launched."""
    try:
        L = hk.load()
    except hk.HIPError:
        pytest.skip("the library is not built")
    def refuses(rc, why):
        assert rc == -1 and why in L.kamd_hip_last_error(), L.kamd_hip_last_error()

    p = 4096    # no pointer: every call is refused before one is used
    quantize, dequantize, gemm = L.kamd_mxfp4_quantize_launch, L.kamd_mxfp4_dequantize_launch, L.kamd_gemm_mxfp4_nt_launch
    refuses(quantize(p, p, p, -1, 32, 32, 1, 0, None), b"bad arguments")
    refuses(quantize(p, p, p, 1, 32, 32, 1, 3, None), b"bad arguments")
    refuses(quantize(p, p, p, 4, 64, 128, 2, 0, None), b"bad arguments")
    refuses(quantize(p, p, p, 1, 1 << 40, 32, 1, 0, None), b"too large")
    refuses(quantize(p, p + 8, p, 4, 64, 64, 1, 0, None), b"aligned")
    for args in ((None, p, p), (p, None, p), (p, p, None)):
        refuses(quantize(*args, 4, 64, 64, 1, 0, None), b"null")
        refuses(dequantize(*args, 4, 64, 0, None), b"null")
    refuses(dequantize(p, p, p, 1, -1, 0, None), b"bad arguments")
    refuses(dequantize(p, p, p, 1, 1, -1, None), b"bad arguments")
    refuses(dequantize(p + 2, p, p, 1, 32, 0, None), b"aligned")
    refuses(gemm(p, p, p, p, p, -1, 1, 1, 1.0, 1, None, 0, None), b"out of range")
    refuses(gemm(p, p, p, p, p, 1, 1 << 40, 1, 1.0, 1, None, 0, None), b"out of range")
    refuses(gemm(p + 8, p, p, p, p, 1, 1, 1, 1.0, 1, None, 0, None), b"aligned")
    for i in range(5):
        refuses(gemm(*[None if j == i else p for j in range(5)], 1, 1, 1, 1.0, 1, None, 0, None), b"null")
    assert gemm(None, None, None, None, None, 0, 1, 1, 1.0, 1, None, 0, None) == 0
    refuses(gemm(p, p, p, p, p, 64, 64, 1024, 1.0, 1, None, 0, None), b"workspace")
    refuses(gemm(p, p, p, p, p, 1, 64, 4096, 1.0, 1, p, 64 * 4, None), b"workspace")
    # where gemm_mxfp4_nt does not ask, none is needed
    for few in (1, 16, 17, 63, 64, 100, 255):
        for many in (1, 64, 255, 256, 1000, 5000, 100000):
            for nb in (1, 7, 8, 63, 256, 500):
                assert L.kamd_gemm_mxfp4_nt_workspace(few, many, nb) == L.kamd_gemm_mxfp4_nt_workspace(many, few, nb) == 0
    need = L.kamd_gemm_mxfp4_nt_workspace(8192, 8192, 256)
    assert need >= 2 * 8192 * 256 and L.kamd_gemm_mxfp4_nt_workspace(1, 8192, 256) == 0
    assert L.kamd_gemm_mxfp4_nt_workspace(-5, 8192, 256) == 0 and L.kamd_gemm_mxfp4_nt_workspace(0, 0, 0) == 0
    for ws, size in ((None, need), (16, need - 1), (8, need)):
        refuses(gemm(p, p, p, p, p, 8192, 8192, 256, 1.0, 1, ws, size, None), b"workspace")
