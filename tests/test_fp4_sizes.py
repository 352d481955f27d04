"""Microscaled fp4 at sizes that one launch does not hold: rows of more than 2^34 values, tall transposed views. Values and
codes are equal, as in the tests of ordinary sizes; between a few written places everything is zero and has to stay so."""
import pytest

torch = pytest.importorskip("torch")

from kubernetes_amd.ops import hip_kernels as hk  # noqa: E402
from test_mxfp4 import operand, quantized, values_of  # noqa: E402


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    hk.load()   # must load: no fallback
    yield torch.device("cuda")
    torch.cuda.empty_cache()


def places(K, edges):
    """Blocks to write around these values of a row and at its ends, as (first, behind the last)."""
    nb = -(-K // 32)
    return [(max(e // 32 - 2, 0), min(e // 32 + 2, nb)) for e in (0, *edges, K)]


def write(x, at, K, seed):
    """Random values at these blocks of each row of x; their codes and scales."""
    g = torch.Generator().manual_seed(seed)
    want = []
    for lo, hi in at:
        v = torch.randn(x.shape[0], min(hi * 32, K) - lo * 32, generator=g).to(x.dtype)
        x[:, lo * 32:lo * 32 + v.shape[1]] = v.to(x.device)
        want.append(quantized(v))
    return want


def nonzero(t):
    """How many are not zero, in pieces: counted at once, a tensor of this size needs several times its memory."""
    return sum(p.count_nonzero().item() for p in t.view(-1).split(1 << 28))


def check(q, s, at, want):
    for (lo, hi), (want_q, want_s) in zip(at, want):
        assert torch.equal(q[:, lo * 16:hi * 16].cpu(), want_q) and torch.equal(s[:, lo:hi].cpu(), want_s)
    assert nonzero(q) == sum(w.count_nonzero().item() for w, _ in want)
    assert nonzero(s) == sum(w.count_nonzero().item() for _, w in want)


@pytest.mark.gpu
def test_quantize_and_dequantize_long_rows(gpu):
    rows, K = 2, (1 << 34) + 37
    at = places(K, [1 << 32, 1 << 33, 3 << 32, 1 << 34])[:-1]
    x = torch.zeros(rows, K, device=gpu, dtype=torch.bfloat16)
    want = write(x, at, K, 1)
    q, s = hk.mxfp4_quantize(x)
    check(q, s, at, want)
    q1, s1 = hk.mxfp4_quantize(x[1])     # one dimension, and an odd start
    assert torch.equal(q1, q[1]) and torch.equal(s1, s[1])
    del q1, s1
    x.fill_(1.0)
    y = hk.mxfp4_dequantize(q, s, k=K)
    total = 0
    for (lo, hi), (want_q, want_s) in zip(at, want):
        v = values_of(want_q, want_s)[:, :min(hi * 32, K) - lo * 32]
        assert torch.equal(y[:, lo * 32:lo * 32 + v.shape[1]].cpu().double(), v)
        total += v.count_nonzero().item()
    assert nonzero(y) == total


@pytest.mark.gpu
def test_dequantize_long_row_to_fp32(gpu):
    K = (1 << 33) + 5
    nb = -(-K // 32)
    q = torch.zeros(1, 16 * nb, device=gpu, dtype=torch.uint8)
    s = torch.full((1, nb), 127, device=gpu, dtype=torch.uint8)
    at = places(K, [1 << 31, 1 << 32])
    for i, (lo, hi) in enumerate(at):
        q[:, lo * 16:hi * 16] = operand(1, hi - lo, i)[0]
    y = hk.mxfp4_dequantize(q, s, k=K, dtype=torch.float32)
    total = 0
    for lo, hi in at:
        v = values_of(q[:, lo * 16:hi * 16], s[:, lo:hi])[:, :min(hi * 32, K) - lo * 32]
        assert torch.equal(y[:, lo * 32:lo * 32 + v.shape[1]].cpu().double(), v)
        total += v.count_nonzero().item()
    assert nonzero(y) == total


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_tall_transposed_view(gpu, dtype):
    rows, K = 2, (1 << 31) + 45
    at = places(K, [1 << 30, (1 << 30) + 4096])
    at[-1] = (at[-1][0] - 1, -(-K // 32))
    x = torch.zeros(K, rows, device=gpu, dtype=dtype).t()
    want = write(x, at, K, 2)
    q, s = hk.mxfp4_quantize(x)
    check(q, s, at, want)


@pytest.mark.gpu
@pytest.mark.parametrize("fp32,dtype", [(True, torch.float32), (False, torch.bfloat16)])
def test_product_over_an_empty_k_behind_32_bits(gpu, fp32, dtype):
    """More than 2^31 outputs, all of them zeros, over memory that held something else."""
    M, N = 46400, 46401
    a, sa = operand(M, 0, 1)
    b, sb = operand(N, 0, 2)
    left = torch.full((M, N), 7.0, device=gpu, dtype=dtype)
    at = left.data_ptr()
    del left
    out = hk.gemm_mxfp4_nt(a, sa, b, sb, out_fp32=fp32)
    assert out.data_ptr() == at and out.shape == (M, N) and out.dtype == dtype
    assert nonzero(out) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,nb", [(1 << 27, 1, 1), (3, 1 << 27, 1), (1, 2, 1 << 27)])
def test_products_of_the_documented_sizes(gpu, M, N, nb):
    """The largest of each size; exact, since what is not zero is little."""
    def sparse(rows, seed):
        q = torch.zeros(rows, 16 * nb, device=gpu, dtype=torch.uint8)
        s = torch.full((rows, nb), 127, device=gpu, dtype=torch.uint8)
        at = sorted({0, 1, rows // 2, rows - 2, rows - 1} & set(range(rows)))
        blocks = sorted({0, 7, nb // 3, nb // 2, nb - 9, nb - 1} & set(range(nb)))
        dense = torch.zeros(len(at), 32 * len(blocks), dtype=torch.float64)
        for i, b in enumerate(blocks):
            pick, scale = operand(len(at), 1, seed + i)
            q[at, b * 16:b * 16 + 16], s[at, b:b + 1] = pick, scale
            dense[:, 32 * i:32 * i + 32] = values_of(pick, scale)
        return q, s, at, dense

    a, sa, at_a, va = sparse(M, 1)
    b, sb, at_b, vb = sparse(N, 50)
    want = (va @ vb.t()).float()
    for fp32, dtype in ((True, torch.float32), (False, torch.bfloat16)):
        out = hk.gemm_mxfp4_nt(a, sa, b, sb, out_fp32=fp32)
        assert torch.equal(out[at_a][:, at_b].cpu(), want.to(dtype))
        assert nonzero(out) == want.count_nonzero().item()


def test_rows_that_no_memory_holds_are_refused():
    try:
        L = hk.load()
    except hk.HIPError:
        pytest.skip("the library is not built")
    p = 4096    # no pointer: every call is refused before one is used
    for K in (1 << 39, 1 << 62):
        for rows in (1, 3):
            for steps in ((K, 1), (1, 2)):
                assert L.kamd_mxfp4_quantize_launch(p, p, p, rows, K, *steps, 0, None) == -1
                assert b"too large" in L.kamd_hip_last_error()
            assert L.kamd_mxfp4_dequantize_launch(p, p, p, rows, K, 2, None) == -1
            assert b"too large" in L.kamd_hip_last_error()


def test_products_past_the_documented_sizes_are_refused():
    try:
        L = hk.load()
    except hk.HIPError:
        pytest.skip("the library is not built")
    p = 4096
    for at in range(3):
        sizes = [1, 1, 1]
        sizes[at] = (1 << 27) + 1
        assert L.kamd_gemm_mxfp4_nt_launch(p, p, p, p, p, *sizes, 1.0, 1, None, 0, None) == -1
        assert b"out of range" in L.kamd_hip_last_error()
