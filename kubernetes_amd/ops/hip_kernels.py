"""ctypes binding for `libkamd_hip.so` (native/hip/kamd_hip.hip, gfx950).

  vector_add(a, b)             -> a + b          (GPU e2e workload kernel)
  gemm_bf16_nt(a, b, out_fp32) -> a @ b.T        (MFMA 16x16x32 bf16, LDS-tiled)
  gemm_fp8_nt(a, b, out_fp32)  -> a @ b.T        (OCP fp8 e4m3, block-scaled MFMA 16x16x128)
  mxfp4_quantize(x)            -> q, scale       (OCP microscaled fp4: e2m1 codes, an e8m0 scale for each 32)
  mxfp4_dequantize(q, scale)   -> x
  gemm_mxfp4_nt(a, a_scale, b, b_scale, out_fp32) -> a @ b.T  (block-scaled MFMA 16x16x128, native/hip/kamd_mxfp4.hip)
  diag_mfma / diag_hbm / diag_vector_add         (device-plugin burn-in diagnostics)
  Payload(dev)                                    (warm per-GPU payload for GPU pods)

The extension is REQUIRED on a GPU host: every entry point raises if the library is missing
rather than silently falling back to a PyTorch implementation.
"""
from __future__ import annotations

import ctypes
import os

from ..native import LIB_DIR

_lib = None


class HIPError(RuntimeError):
    pass


def lib_path():
    return os.path.join(LIB_DIR, "libkamd_hip.so")


def load():
    global _lib
    if _lib is None:
        p = lib_path()
        if not os.path.exists(p):
            raise HIPError(f"{p} is not built (python -m kubernetes_amd.native.build); no fallback exists")
        L = ctypes.CDLL(p)
        vp, i, f, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
        L.kamd_hip_last_error.restype = ctypes.c_char_p
        L.kamd_vector_add_launch.argtypes = [vp, vp, vp, i, vp]
        L.kamd_gemm_bf16_nt_launch.argtypes = [vp, vp, vp, i, i, i, i, f, i, vp]
        L.kamd_gemm_fp8_nt_launch.argtypes = [vp, vp, vp, i, i, i, i, f, i, vp]
        i64 = ctypes.c_int64
        L.kamd_mxfp4_quantize_launch.argtypes = [vp, vp, vp, i64, i64, i64, i64, i, vp]
        L.kamd_mxfp4_dequantize_launch.argtypes = [vp, vp, vp, i64, i64, i, vp]
        L.kamd_gemm_mxfp4_nt_launch.argtypes = [vp, vp, vp, vp, vp, i64, i64, i64, f, i, vp, i64, vp]
        L.kamd_gemm_mxfp4_nt_workspace.argtypes = [i64, i64, i64]
        L.kamd_gemm_mxfp4_nt_workspace.restype = i64
        L.kamd_hbm_copy_launch.argtypes = [vp, vp, sz, vp]
        L.kamd_diag_vector_add.argtypes = [i, i, ctypes.POINTER(ctypes.c_float)]
        L.kamd_diag_mfma.argtypes = [i, i, i, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)]
        L.kamd_diag_mfma_fp8.argtypes = [i, i, i, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)]
        L.kamd_diag_mfma_fp4.argtypes = [i, i, i, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)]
        L.kamd_diag_vector_add_error.argtypes = [vp, vp, vp, i]
        L.kamd_diag_vector_add_error.restype = f
        L.kamd_diag_mfma_sample.argtypes = [vp, vp, i, i, f, ctypes.POINTER(ctypes.c_double)]
        L.kamd_diag_mfma_sample.restype = None
        L.kamd_diag_mfma_fp4_sample.argtypes = [vp, vp, vp, vp, vp, vp, i, f, ctypes.POINTER(ctypes.c_double)]
        L.kamd_diag_hbm.argtypes = [i, sz, i, ctypes.POINTER(ctypes.c_double)]
        L.kamd_payload_create.argtypes = [i, i]
        L.kamd_payload_create.restype = vp
        L.kamd_payload_run.argtypes = [vp]
        L.kamd_payload_run_batch.argtypes = [vp, i, ctypes.POINTER(ctypes.c_int)]
        L.kamd_payload_destroy.argtypes = [vp]
        L.kamd_hip_device_arch.argtypes = [i, ctypes.c_char_p, i]
        L.kamd_gemm_set_path.argtypes = [i]
        L.kamd_gemm_set_group.argtypes = [i]
        L.kamd_hbm_copy_config.argtypes = [i, i]
        _lib = L
    return _lib


def _raise(rc, what):
    if rc != 0:
        raise HIPError(f"{what}: {load().kamd_hip_last_error().decode(errors='replace')}")


def _stream(t):
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def device_count() -> int:
    return load().kamd_hip_device_count()


def device_arch(dev=0) -> str:
    buf = ctypes.create_string_buffer(64)
    _raise(load().kamd_hip_device_arch(dev, buf, 64), "device_arch")
    return buf.value.decode()


def vector_add(a, b):
    import torch
    assert a.is_cuda and a.dtype == torch.float32 and a.shape == b.shape and a.is_contiguous() and b.is_contiguous()
    out = torch.empty_like(a)
    _raise(load().kamd_vector_add_launch(a.data_ptr(), b.data_ptr(), out.data_ptr(), a.numel(), _stream(a)), "vector_add")
    return out


def gemm_bf16_nt(a, b, out_fp32=True, alpha=1.0):
    """C = alpha * a @ b.T with a: [M, K] bf16, b: [N, K] bf16 (both row-major, K % 8 == 0)."""
    import torch
    assert a.is_cuda and b.is_cuda and a.dtype == torch.bfloat16 and b.dtype == torch.bfloat16
    assert a.dim() == 2 and b.dim() == 2 and a.shape[1] == b.shape[1], (a.shape, b.shape)
    a, b = a.contiguous(), b.contiguous()
    M, K = a.shape
    N = b.shape[0]
    if K % 8:
        raise ValueError(f"K={K} must be a multiple of 8")
    out = torch.empty((M, N), device=a.device, dtype=torch.float32 if out_fp32 else torch.bfloat16)
    _raise(load().kamd_gemm_bf16_nt_launch(a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K, N, float(alpha),
                                           1 if out_fp32 else 0, _stream(a)), "gemm_bf16_nt")
    return out


def gemm_fp8_nt(a, b, out_fp32=True, alpha=1.0):
    """C = alpha * a @ b.T with a: [M, K], b: [N, K] OCP fp8 e4m3 (torch.float8_e4m3fn), fp32
    accumulate, on the block-scaled MFMA (v_mfma_scale_f32_16x16x128_f8f6f4, unit scales).
    M, N must be multiples of 256 and K of 128."""
    import torch
    assert a.is_cuda and b.is_cuda and a.dtype == torch.float8_e4m3fn and b.dtype == torch.float8_e4m3fn
    assert a.dim() == 2 and b.dim() == 2 and a.shape[1] == b.shape[1], (a.shape, b.shape)
    a, b = a.contiguous(), b.contiguous()
    M, K = a.shape
    N = b.shape[0]
    if M % 256 or N % 256 or K % 128:
        raise ValueError(f"gemm_fp8_nt needs M, N % 256 == 0 and K % 128 == 0, got {M}x{N}x{K}")
    out = torch.empty((M, N), device=a.device, dtype=torch.float32 if out_fp32 else torch.bfloat16)
    _raise(load().kamd_gemm_fp8_nt_launch(a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K, N, float(alpha),
                                          1 if out_fp32 else 0, _stream(a)), "gemm_fp8_nt")
    return out


MXFP4_BLOCK = 32
_mx_type_codes = {}


def _mx_types():
    """The C entries' codes of the types that fp4 is made from and turned into."""
    if not _mx_type_codes:
        import torch
        _mx_type_codes.update({torch.bfloat16: 0, torch.float16: 1, torch.float32: 2})
    return _mx_type_codes


def _mx_launch(index, what, entry, *args):
    """A launch on the current stream of that device, whichever device is current."""
    import torch
    cuda = torch._C   # what torch.cuda.current_device and current_stream ask, 2 us sooner
    if index == cuda._cuda_getDevice():
        rc = entry(*args, cuda._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = entry(*args, cuda._cuda_getCurrentRawStream(index))
    if rc:
        _raise(rc, what)


def _mx_pair(q, scale, what):
    """Codes and scales as contiguous bytes, `q` 16-byte aligned: as they are where they are so already."""
    import torch
    u8 = torch.uint8
    qs, ss = q.shape, scale.shape
    if (len(qs) == 2 == len(ss) and q.dtype is u8 is scale.dtype and qs[0] == ss[0] and qs[1] == 16 * ss[1]
            and q.is_contiguous() and scale.is_contiguous() and q.get_device() == scale.get_device() >= 0
            and not q.data_ptr() % 16):
        return q, scale
    if q.dtype not in (u8, torch.float4_e2m1fn_x2):
        raise ValueError(f"{what}: codes must be uint8 or float4_e2m1fn_x2, got {q.dtype}")
    if scale.dtype not in (u8, torch.float8_e8m0fnu):
        raise ValueError(f"{what}: scales must be uint8 or float8_e8m0fnu, got {scale.dtype}")
    if not qs or len(qs) != len(ss) or qs[-1] != 16 * ss[-1] or qs[:-1] != ss[:-1]:
        raise ValueError(f"{what}: codes [..., 16 * blocks] need scales [..., blocks], got {tuple(qs)} and {tuple(ss)}")
    if q.device != scale.device:
        raise ValueError(f"{what}: codes on {q.device}, scales on {scale.device}")
    if q.dtype is not u8:
        q = q.view(u8)
    if scale.dtype is not u8:
        scale = scale.view(u8)
    q, scale = q.contiguous(), scale.contiguous()
    return q.clone() if q.data_ptr() % 16 else q, scale


def _mx_gpu(t, what):
    """The index of the tensor's GPU."""
    index = t.get_device()
    if index < 0 or not t.is_cuda:
        raise ValueError(f"{what} needs tensors on the GPU, got {t.device}")
    return index


def mxfp4_quantize(x):
    """x [..., K] (bf16, fp16 or fp32, any strides) as microscaled fp4: codes [..., 16 * nb] and scales
    [..., nb], both uint8, nb = ceil(K / 32).

    32 values along the last axis share the scale 2^(s - 127), s = floor(log2(max |x|)) - 2 + 127 and 0 at
    least; each value is rounded to the nearest of 0 0.5 1 1.5 2 3 4 6 times it (ties to the even code, 6 at
    most). The lower index is in the low nibble; a last short block is filled with zeros. A block that holds
    a NaN or an infinity gets s = 255: all of it stands for NaN. No gradient is recorded."""
    import torch
    code = _mx_types().get(x.dtype)
    if code is None:
        raise ValueError(f"mxfp4_quantize needs bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("mxfp4_quantize needs at least one dimension")
    index = _mx_gpu(x, "mxfp4_quantize")
    *lead, K = x.shape
    nb = -(-K // MXFP4_BLOCK)
    if len(lead) == 1 and nb:   # strides given: a quarter of a microsecond sooner each
        rows, u8, dev = lead[0], torch.uint8, x.device
        q = torch.empty_strided((rows, 16 * nb), (16 * nb, 1), dtype=u8, device=dev)
        scale = torch.empty_strided((rows, nb), (nb, 1), dtype=u8, device=dev)
    else:
        q = x.new_empty((*lead, 16 * nb), dtype=torch.uint8)
        scale = x.new_empty((*lead, nb), dtype=torch.uint8)
    if K == 0 or 0 in lead:
        return q, scale
    x2 = x if len(lead) == 1 else x.reshape(-1, K)
    if x2.is_neg():   # a view whose values are the negated ones of memory
        x2 = x2.resolve_neg()
    row_step, step = x2.stride()
    if K > 1 and step != 1 and row_step != 1:   # neither rows nor columns in one piece each
        x2 = x2.contiguous()
        row_step, step = K, 1
    _mx_launch(index, "mxfp4_quantize", load().kamd_mxfp4_quantize_launch, x2.data_ptr(), q.data_ptr(), scale.data_ptr(),
               x2.shape[0], K, row_step, step, code)
    return q, scale


def mxfp4_dequantize(q, scale, k=None, dtype=None):
    """The values [..., k] that microscaled fp4 codes [..., 16 * nb] and scales [..., nb] stand for, rounded
    once to `dtype` (bf16 unless given; fp16, fp32). `k` leaves out what fills the last block; 32 * nb unless
    given. Scale 255 gives NaN. Codes and scales are uint8 or torch's float4_e2m1fn_x2 and float8_e8m0fnu."""
    import torch
    dtype = torch.bfloat16 if dtype is None else dtype
    code = _mx_types().get(dtype)
    if code is None:
        raise ValueError(f"mxfp4_dequantize gives bf16, fp16 or fp32, not {dtype}")
    q, scale = _mx_pair(q, scale, "mxfp4_dequantize")
    *lead, nb = scale.shape
    k = MXFP4_BLOCK * nb if k is None else int(k)
    if k < 0 or -(-k // MXFP4_BLOCK) != nb:
        raise ValueError(f"mxfp4_dequantize: k={k} does not have {nb} blocks of {MXFP4_BLOCK}")
    index = _mx_gpu(q, "mxfp4_dequantize")
    if len(lead) == 1 and k:
        x = torch.empty_strided((lead[0], k), (k, 1), dtype=dtype, device=q.device)
    else:
        x = q.new_empty((*lead, k), dtype=dtype)
    if k == 0 or 0 in lead:
        return x
    _mx_launch(index, "mxfp4_dequantize", load().kamd_mxfp4_dequantize_launch, q.data_ptr(), scale.data_ptr(), x.data_ptr(),
               scale.numel() // nb, k, code)
    return x


def gemm_mxfp4_nt(a, a_scale, b, b_scale, out_fp32=True, alpha=1.0):
    """C = alpha * a @ b.T of microscaled fp4 operands as mxfp4_quantize makes them: a [M, 16 * nb], a_scale
    [M, nb], b [N, 16 * nb], b_scale [N, nb]; sums in fp32, C fp32 or bf16. Any M, N and nb up to 2^27 each; K is
    32 * nb. A block of scale 255 makes every output that it enters NaN. No gradient is recorded."""
    import torch
    sa, sb = a.shape, b.shape
    if len(sa) != 2 or len(sb) != 2 or sa[1] != sb[1]:
        raise ValueError(f"gemm_mxfp4_nt needs codes [M, 16 * blocks] and [N, 16 * blocks], got {tuple(sa)} and {tuple(sb)}")
    if a.get_device() != b.get_device():
        raise ValueError(f"gemm_mxfp4_nt: a on {a.device}, b on {b.device}")
    a, a_scale = _mx_pair(a, a_scale, "gemm_mxfp4_nt a")
    b, b_scale = _mx_pair(b, b_scale, "gemm_mxfp4_nt b")
    index = _mx_gpu(a, "gemm_mxfp4_nt")
    M, N, nb = sa[0], sb[0], sa[1] // 16
    L = load()
    out = torch.empty_strided((M, N), (N or 1, 1), dtype=torch.float32 if out_fp32 else torch.bfloat16, device=a.device)
    # none for few rows, but of a long K
    need = L.kamd_gemm_mxfp4_nt_workspace(M, N, nb) if nb > 500 or (M >= 256 and N >= 256) else 0
    ws = torch.empty(need, dtype=torch.uint8, device=a.device) if need else None
    _mx_launch(index, "gemm_mxfp4_nt", L.kamd_gemm_mxfp4_nt_launch, a.data_ptr(), a_scale.data_ptr(), b.data_ptr(),
               b_scale.data_ptr(), out.data_ptr(), M, N, nb, float(alpha), 1 if out_fp32 else 0,
               ws.data_ptr() if need else None, need)
    return out


def set_gemm_group(group: int):
    """M-tiles per group of the ping-pong GEMM's L2-friendly tile order (default 4)."""
    load().kamd_gemm_set_group(int(group))


def set_gemm_path(path: int):
    """0 = auto (the ping-pong 256x256 global_load_lds kernel — wave groups staggered by one
    barrier — when M, N % 256 == 0 and K % 64 == 0, else the 128x128 kernel), 1 = always the
    128x128 register-staged kernel, 2 = the 2-barrier 256x256 kernel, 3 = ping-pong, 4-6 =
    ping-pong variants (LDS epilogue / static priority / both), 7 = the 8-phase 256x256 kernel."""
    load().kamd_gemm_set_path(int(path))


def hbm_copy_config(variant: int = 0, blocks: int = 0):
    """variant 0: flat, one 16-B element per lane (default, ~6.2 TB/s); 1: grid-stride;
    2: 4 non-temporal loads in flight per lane; 3: the same without the hints."""
    load().kamd_hbm_copy_config(int(variant), int(blocks))


def hbm_copy(src, dst):
    assert src.is_cuda and dst.is_cuda and src.numel() * src.element_size() == dst.numel() * dst.element_size()
    nbytes = src.numel() * src.element_size()
    assert nbytes % 16 == 0
    _raise(load().kamd_hbm_copy_launch(src.data_ptr(), dst.data_ptr(), nbytes, _stream(src)), "hbm_copy")


def diag_vector_add(dev=0, n=50000) -> float:
    e = ctypes.c_float()
    _raise(load().kamd_diag_vector_add(dev, n, ctypes.byref(e)), "diag_vector_add")
    return e.value


def diag_mfma(dev=0, size=4096, iters=20):
    tf, err = ctypes.c_double(), ctypes.c_double()
    _raise(load().kamd_diag_mfma(dev, size, iters, ctypes.byref(tf), ctypes.byref(err)), "diag_mfma")
    return {"tflops": tf.value, "max_rel_err": err.value, "size": size, "iters": iters}


def diag_mfma_fp8(dev=0, size=8192, iters=10):
    tf, err = ctypes.c_double(), ctypes.c_double()
    _raise(load().kamd_diag_mfma_fp8(dev, size, iters, ctypes.byref(tf), ctypes.byref(err)), "diag_mfma_fp8")
    return {"tflops": tf.value, "max_rel_err": err.value, "size": size, "iters": iters}


def diag_mfma_fp4(dev=0, size=8192, iters=10):
    """Quantises random bf16 operands to microscaled fp4 and multiplies them; a code or scale that is not the
    definition's makes `max_rel_err` 1, an output that is NaN makes it infinite."""
    tf, err = ctypes.c_double(), ctypes.c_double()
    _raise(load().kamd_diag_mfma_fp4(dev, size, iters, ctypes.byref(tf), ctypes.byref(err)), "diag_mfma_fp4")
    return {"tflops": tf.value, "max_rel_err": err.value, "size": size, "iters": iters}


def diag_hbm(dev=0, nbytes=1 << 30, iters=20):
    g = ctypes.c_double()
    _raise(load().kamd_diag_hbm(dev, nbytes, iters, ctypes.byref(g)), "diag_hbm")
    return {"GBps": g.value, "bytes": nbytes, "iters": iters}


class Payload:
    """Warm per-GPU context: `run()` launches vector_add on the device and verifies it."""

    def __init__(self, dev=0, n=50000):
        self.h = load().kamd_payload_create(dev, n)
        if not self.h:
            raise HIPError(f"payload create on device {dev} failed")
        self.dev = dev

    MAX_BATCH = 256   # PAYLOAD_SLOTS in native/hip/kamd_hip.hip

    def run(self) -> bool:
        return load().kamd_payload_run(self.h) == 0

    def run_batch(self, k: int) -> list:
        """k container starts at once: k vector_add launches, one verify kernel, one sync.
        Returns one pass/fail per start. Thread-safe for a single caller thread at a time."""
        out = []
        while k > 0:
            m = min(k, self.MAX_BATCH)
            ok = (ctypes.c_int * m)()
            rc = load().kamd_payload_run_batch(self.h, m, ok)
            out += [False] * m if rc < 0 else [bool(x) for x in ok]
            k -= m
        return out

    def close(self):
        if self.h:
            load().kamd_payload_destroy(self.h)
            self.h = None
