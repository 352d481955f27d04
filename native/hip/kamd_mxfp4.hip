// kamd_mxfp4 — microscaled 4-bit floating point on gfx950: quantisation, its inverse, and the product.
//
// Format (OCP microscaling 1.0): 32 consecutive values of a row form a block; each is an e2m1 code
// (sign, 0 0.5 1 1.5 2 3 4 6) times the block's e8m0 scale 2^(s - 127); s = 255 is NaN.
// Layout: nb = ceil(K / 32) blocks a row; codes q[row][16 * nb] bytes, the lower index in the low nibble,
// zero codes behind K; scales scale[row][nb] bytes. A row is whole 16-byte chunks, one a block, whatever
// K is, so no kernel below meets a code that straddles a row.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <new>
#include <vector>

#include "kamd_hip_err.h"

#define HC(x)                                 \
  do {                                        \
    if (kamd_check((x), #x) != 0) return -1;  \
  } while (0)

namespace mxfp4 {
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

enum Type { BF16 = 0, FP16 = 1, FP32 = 2 };   // the C entries' type codes
template <int TYPE> struct Elem { typedef uint16_t bits; };
template <> struct Elem<FP32> { typedef uint32_t bits; };

// ---------------------------------------------------------------------------
// Quantisation: amax = max |x| of the block, s = max(floor(log2 amax) - 2 + 127, 0), code = x / 2^(s - 127)
// rounded to e2m1 (nearest, ties to the even code, 6 at most). floor(log2) is the exponent field of amax,
// read as fp32: exact for fp16's subnormals, and 0 for fp32's own, whose blocks have s = 0 either way.
// The rounding is v_cvt_scalef32_pk_fp4_*: it rounds and saturates as above for every value and scale,
// subnormals among them. It has no answer for infinities and NaN; a block that holds one gets s = 255.

// 8 consecutive values of one lane; 4 neighbouring lanes hold a block. The maximum is taken over the bits
// of |x| as integers: their order is that of the values, and NaN is above infinity.
template <int TYPE> struct Oct;
template <> struct Oct<FP32> {
  uint32_t v[8];
  __device__ uint32_t amax() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, v[i] & 0x7fffffffu);
    return m;
  }
  __device__ uint32_t codes(float scale) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[0]), __uint_as_float(v[1]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[2]), __uint_as_float(v[3]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[4]), __uint_as_float(v[5]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[6]), __uint_as_float(v[7]), scale, 3);
    return c;
  }
};
struct Oct16 {
  uint32_t v[4];   // pairs
  __device__ uint32_t amax16() const {
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
    return max((uint32_t)m.x, (uint32_t)m.y);
  }
};
template <> struct Oct<BF16> : Oct16 {
  __device__ uint32_t amax() const { return amax16() << 16; }
  __device__ uint32_t codes(float scale) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, v[0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, v[1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, v[2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, v[3]), scale, 3);
    return c;
  }
};
template <> struct Oct<FP16> : Oct16 {
  __device__ uint32_t amax() const {
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)amax16()));
  }
  __device__ uint32_t codes(float scale) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, v[0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, v[1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, v[2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, v[3]), scale, 3);
    return c;
  }
};

__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255 ? 255u : max(e, 2u) - 2;
}

// Item i is 8 values: row i / (4 nb), values 8 (i % (4 nb)) .. + 7 of it. Codes and scales are written as
// one run: item i's codes at byte 4 i, block i / 4's scale at byte i / 4.
template <int TYPE>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const void* __restrict__ xv, uint32_t* __restrict__ q, uint8_t* __restrict__ scale,
                     size_t first, size_t items, uint32_t row_items, int64_t K, int64_t ld) {
  typedef typename Elem<TYPE>::bits bits;
  const size_t base = first + (size_t)blockIdx.x * 256;   // uniform: one 64-bit division a workgroup
  const size_t i = base + threadIdx.x;
  if (i >= items) return;
  const size_t row0 = base / row_items;
  const uint32_t at = (uint32_t)(base - row0 * row_items) + threadIdx.x, over = at / row_items;
  const int64_t k0 = (int64_t)(at - over * row_items) * 8;
  const bits* p = (const bits*)xv + (int64_t)(row0 + over) * ld + k0;
  Oct<TYPE> o;
  if (k0 + 8 <= K) {
    __builtin_memcpy(&o, p, sizeof o);
  } else {
    bits t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = k0 + j < K ? p[j] : (bits)0;
    __builtin_memcpy(&o, t, sizeof o);
  }
  uint32_t m = o.amax();
  m = max(m, (uint32_t)__shfl_xor((int)m, 1));
  m = max(m, (uint32_t)__shfl_xor((int)m, 2));
  const uint32_t s = scale_byte(m);
  q[i] = s == 255 ? 0u : o.codes(__uint_as_float(s << 23));
  if ((threadIdx.x & 3) == 0) scale[i >> 2] = (uint8_t)s;
}

// The inverse, rounded once to the output's type. v_cvt_scalef32_pk_*_fp4 gives NaN for s = 255.
template <int TYPE>
__global__ void __launch_bounds__(256)
dequantize_kernel(const uint32_t* __restrict__ q, const uint8_t* __restrict__ scale, void* __restrict__ xv,
                  size_t first, size_t items, uint32_t row_items, int64_t K) {
  typedef typename Elem<TYPE>::bits bits;
  const size_t base = first + (size_t)blockIdx.x * 256;
  const size_t i = base + threadIdx.x;
  if (i >= items) return;
  const size_t row0 = base / row_items;
  const uint32_t at = (uint32_t)(base - row0 * row_items) + threadIdx.x, over = at / row_items;
  const int64_t k0 = (int64_t)(at - over * row_items) * 8;
  const uint32_t c = q[i];
  const float s = __uint_as_float((uint32_t)scale[i >> 2] << 23);
  bits t[8];
  if constexpr (TYPE == FP32) {
    const f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3)};
    __builtin_memcpy(t, v, sizeof t);
  } else if constexpr (TYPE == BF16) {
    const bf16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3)};
    __builtin_memcpy(t, v, sizeof t);
  } else {
    const f16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 3)};
    __builtin_memcpy(t, v, sizeof t);
  }
  bits* p = (bits*)xv + (int64_t)(row0 + over) * K + k0;
  if (k0 + 8 <= K) {
    __builtin_memcpy(p, t, sizeof t);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k0 + j < K) p[j] = t[j];
  }
}

// ---------------------------------------------------------------------------
// Product C[M, N] = alpha * A[M, K] B[N, K]^T on v_mfma_scale_f32_16x16x128_f8f6f4, sums in fp32.
//
// One instruction takes 16 rows x 128 values of each operand: lane l holds the 16-byte chunk (one block)
// l >> 4 of row l & 15 and, as a byte, that block's scale. Which 4 chunks of K a step takes is free as long
// as both operands take the same ones.

__device__ __forceinline__ i32x8 frag(i32x4 v) { return i32x8{v.x, v.y, v.z, v.w, 0, 0, 0, 0}; }

__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_out(__bf16* p, float v) { *p = (__bf16)v; }

// One 16x16 tile a workgroup; its 4 waves take the steps of K in turn and join their sums in LDS.
// Rows behind the last are read as the last row and not stored. Chunks behind the last block are read as
// the row's last block, with their codes cleared and the scale set to 1 on both sides.
constexpr int SMALL_WAVES = 4;
template <typename OutT>
__global__ void __launch_bounds__(SMALL_WAVES * 64)
gemm_small_kernel(const uint8_t* __restrict__ A, const uint8_t* __restrict__ As, const uint8_t* __restrict__ B,
                  const uint8_t* __restrict__ Bs, OutT* __restrict__ C, int M, int N, int nb, float alpha) {
  __shared__ f32x4 part[SMALL_WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int tiles_n = (N + 15) / 16;
  const int m0 = (int)(blockIdx.x / tiles_n) * 16, n0 = (int)(blockIdx.x % tiles_n) * 16;
  const size_t ra = (size_t)min(m0 + r, M - 1) * nb, rb = (size_t)min(n0 + r, N - 1) * nb;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = wave * 4; c0 < nb; c0 += SMALL_WAVES * 4) {
    const int c = min(c0 + g, nb - 1);
    i32x4 a = *(const i32x4*)(A + (ra + c) * 16), b = *(const i32x4*)(B + (rb + c) * 16);
    int sa = As[ra + c], sb = Bs[rb + c];
    if (c0 + g >= nb) {
      a = b = i32x4{0, 0, 0, 0};
      sa = sb = 127;
    }
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(frag(a), frag(b), acc, 4, 4, 0, sa, 0, sb);
  }
  part[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < SMALL_WAVES; ++w) acc += part[w][lane];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = m0 + g * 4 + j, col = n0 + r;
    if (row < M && col < N) store_out(C + (size_t)row * N + col, alpha * acc[j]);
  }
}

template <typename OutT>
__global__ void __launch_bounds__(256) zero_kernel(OutT* __restrict__ C, size_t n) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) C[i] = (OutT)0.f;
}

// A launch's workgroups times 256 lanes stay below 2^32; longer runs take several launches.
constexpr size_t SLICE = (size_t)1 << 31;

template <typename F>
static int sliced(size_t items, const char* what, F launch) {
  for (size_t first = 0; first < items; first += SLICE) {
    const size_t n = items - first < SLICE ? items - first : SLICE;
    launch(first, dim3((unsigned)((n + 255) / 256)));
    HC(hipGetLastError());
  }
  (void)what;
  return 0;
}
}  // namespace mxfp4

extern "C" {

// x: rows of K values (type 0 bf16, 1 fp16, 2 fp32), row r at x + r * ld elements; q: rows * 16 * nb bytes, 4-byte
// aligned; scale: rows * nb bytes
int kamd_mxfp4_quantize_launch(const void* x, void* q, void* scale, int64_t rows, int64_t K, int64_t ld, int type,
                               hipStream_t stream) {
  if (rows < 0 || K < 0 || type < 0 || type > 2) return kamd_fail("mxfp4_quantize: bad arguments");
  if (rows == 0 || K == 0) return 0;
  const int64_t row_items = (K + 31) / 32 * 4;
  if (row_items >= (int64_t)1 << 31) return kamd_fail("mxfp4_quantize: K (%lld) is too large", (long long)K);
  const size_t items = (size_t)rows * row_items;
  return mxfp4::sliced(items, "mxfp4_quantize", [&](size_t first, dim3 grid) {
    auto k = type == mxfp4::BF16   ? mxfp4::quantize_rows_kernel<mxfp4::BF16>
             : type == mxfp4::FP16 ? mxfp4::quantize_rows_kernel<mxfp4::FP16>
                                   : mxfp4::quantize_rows_kernel<mxfp4::FP32>;
    hipLaunchKernelGGL(k, grid, dim3(256), 0, stream, x, (uint32_t*)q, (uint8_t*)scale, first, items,
                       (uint32_t)row_items, K, ld);
  });
}

// the inverse into contiguous rows of K values; q is 4-byte aligned
int kamd_mxfp4_dequantize_launch(const void* q, const void* scale, void* x, int64_t rows, int64_t K, int type,
                                 hipStream_t stream) {
  if (rows < 0 || K < 0 || type < 0 || type > 2) return kamd_fail("mxfp4_dequantize: bad arguments");
  if (rows == 0 || K == 0) return 0;
  const int64_t row_items = (K + 31) / 32 * 4;
  if (row_items >= (int64_t)1 << 31) return kamd_fail("mxfp4_dequantize: K (%lld) is too large", (long long)K);
  const size_t items = (size_t)rows * row_items;
  return mxfp4::sliced(items, "mxfp4_dequantize", [&](size_t first, dim3 grid) {
    auto k = type == mxfp4::BF16   ? mxfp4::dequantize_kernel<mxfp4::BF16>
             : type == mxfp4::FP16 ? mxfp4::dequantize_kernel<mxfp4::FP16>
                                   : mxfp4::dequantize_kernel<mxfp4::FP32>;
    hipLaunchKernelGGL(k, grid, dim3(256), 0, stream, (const uint32_t*)q, (const uint8_t*)scale, x, first, items,
                       (uint32_t)row_items, K);
  });
}

// C[M, N] = alpha * A B^T, A [M, 16 nb] / As [M, nb], B [N, 16 nb] / Bs [N, nb] contiguous, A and B 16-byte aligned;
// C fp32 or bf16, contiguous. nb = 0 gives zeros.
int kamd_gemm_mxfp4_nt_launch(const void* A, const void* As, const void* B, const void* Bs, void* C, int64_t M, int64_t N,
                              int64_t nb, float alpha, int out_fp32, hipStream_t stream) {
  using namespace mxfp4;
  const int64_t most = (int64_t)1 << 27;
  if (M < 0 || N < 0 || nb < 0 || M > most || N > most || nb > most)
    return kamd_fail("gemm_mxfp4_nt: sizes out of range (%lld x %lld x %lld blocks)", (long long)M, (long long)N, (long long)nb);
  if (M == 0 || N == 0) return 0;
  if ((((uintptr_t)A) | ((uintptr_t)B)) & 15) return kamd_fail("gemm_mxfp4_nt: A/B must be 16-byte aligned");
  if (nb == 0) {
    const size_t n = (size_t)M * N;
    if (n > SLICE) return kamd_fail("gemm_mxfp4_nt: an empty K with more than 2^31 outputs");
    if (out_fp32)
      hipLaunchKernelGGL(zero_kernel<float>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, (float*)C, n);
    else
      hipLaunchKernelGGL(zero_kernel<__bf16>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, (__bf16*)C, n);
    return kamd_check(hipGetLastError(), "gemm_mxfp4_nt launch");
  }
  const int64_t tiles = ((M + 15) / 16) * ((N + 15) / 16);
  if (tiles * (SMALL_WAVES * 64) >= (int64_t)1 << 32) return kamd_fail("gemm_mxfp4_nt: %lld x %lld is too large", (long long)M, (long long)N);
  if (out_fp32)
    hipLaunchKernelGGL(gemm_small_kernel<float>, dim3((unsigned)tiles), dim3(SMALL_WAVES * 64), 0, stream, (const uint8_t*)A,
                       (const uint8_t*)As, (const uint8_t*)B, (const uint8_t*)Bs, (float*)C, (int)M, (int)N, (int)nb, alpha);
  else
    hipLaunchKernelGGL(gemm_small_kernel<__bf16>, dim3((unsigned)tiles), dim3(SMALL_WAVES * 64), 0, stream, (const uint8_t*)A,
                       (const uint8_t*)As, (const uint8_t*)B, (const uint8_t*)Bs, (__bf16*)C, (int)M, (int)N, (int)nb, alpha);
  return kamd_check(hipGetLastError(), "gemm_mxfp4_nt launch");
}

}  // extern "C"
