// kamd_mxfp4 — microscaled 4-bit floating point on gfx950: quantisation, its inverse, and the product.
//
// Format (OCP microscaling 1.0): 32 consecutive values of a row form a block; each is an e2m1 code
// (sign, 0 0.5 1 1.5 2 3 4 6) times the block's e8m0 scale 2^(s - 127); s = 255 is NaN.
// Layout: nb = ceil(K / 32) blocks a row; codes q[row][16 * nb] bytes, the lower index in the low nibble,
// zero codes behind K; scales scale[row][nb] bytes. A row is whole 16-byte chunks, one a block, whatever
// K is, so no kernel below meets a code that straddles a row.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include <atomic>
#include <cmath>
#include <exception>
#include <type_traits>
#include <utility>
#include <vector>

#include "kamd_diag.h"
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
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));   // where values of 2 bytes may lie
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
// |x| of a 16-bit type as the bits of an fp32
template <int TYPE>
__device__ __forceinline__ uint32_t widen(uint32_t v) {
  if constexpr (TYPE == BF16) return v << 16;
  else return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)v));
}
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
  __device__ uint32_t amax() const { return widen<BF16>(amax16()); }
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
  __device__ uint32_t amax() const { return widen<FP16>(amax16()); }
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
  const uint32_t c = s == 255 ? 0u : o.codes(__uint_as_float(s << 23));
  // past the caches: 8192x8192 from fp32 42 against 49 us, but from bf16 31 against 28
  if constexpr (TYPE == FP32) __builtin_nontemporal_store(c, q + i);
  else q[i] = c;
  if ((threadIdx.x & 3) == 0) scale[i >> 2] = (uint8_t)s;
}

// The same of x whose columns lie in one piece each (a transposed view): value k of row m at x[k * ld + m]. A wave
// reads 32 rows of memory, 256 bytes of each, a lane having all 32 values of COLS blocks; 8 blocks of a row go
// through LDS, so that whole cache lines are written. Rows of memory and columns behind the last read as 0.
template <int TYPE>
__global__ void __launch_bounds__(512)
quantize_cols_kernel(const void* __restrict__ xv, uint8_t* __restrict__ q, uint8_t* __restrict__ scale, int64_t first, int64_t M,
                     int64_t K, int64_t ld, int64_t nb) {
  typedef typename Elem<TYPE>::bits bits;
  constexpr int COLS = TYPE == FP32 ? 1 : 2, ROWS = 64 * COLS, PITCH = 128 + 16;
  __shared__ __attribute__((aligned(16))) uint8_t codes[ROWS * PITCH];
  __shared__ __attribute__((aligned(8))) uint8_t scales[ROWS * 8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t tiles_m = (M + ROWS - 1) / ROWS, tile = first + blockIdx.x;
  const int64_t m0 = tile % tiles_m * ROWS, b0 = tile / tiles_m * 8;
  const int64_t m = m0 + lane * COLS;
  {
    const int b = wave;
    const int64_t k0 = (b0 + b) * 32;
    const bits* p = (const bits*)xv + k0 * ld + m;
    uint32_t v[32];
    const int ks = (int)(K - k0 < 32 ? K - k0 : 32);   // <= 0: no block
    if (ks == 32 && m + COLS <= M) {
#pragma unroll
      for (int k = 0; k < 32; ++k) __builtin_memcpy(&v[k], p + k * ld, 4);
    } else {
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        v[k] = 0;
#pragma unroll
        for (int c = 0; c < COLS; ++c)
          if (k < ks && m + c < M) v[k] |= (uint32_t)p[k * ld + c] << (16 * c);
      }
    }
    // each column's codes as those of 4 lanes of the kernel above
    uint32_t amax[COLS];
    if constexpr (TYPE == FP32) {
      amax[0] = 0;
#pragma unroll
      for (int k = 0; k < 32; ++k) amax[0] = max(amax[0], v[k] & 0x7fffffffu);
    } else {
      u16x2 a = {0, 0};
#pragma unroll
      for (int k = 0; k < 32; ++k) a = __builtin_elementwise_max(a, __builtin_bit_cast(u16x2, v[k] & 0x7fff7fffu));
      amax[0] = widen<TYPE>(a.x);
      amax[1] = widen<TYPE>(a.y);
    }
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const uint32_t s = scale_byte(amax[c]);
      uint32_t out[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        Oct<TYPE> o;
        if constexpr (TYPE == FP32) {
#pragma unroll
          for (int k = 0; k < 8; ++k) o.v[k] = v[i * 8 + k];
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            o.v[k] = __builtin_amdgcn_perm(v[i * 8 + k * 2 + 1], v[i * 8 + k * 2], c == 0 ? 0x05040100u : 0x07060302u);
        }
        out[i] = s == 255 ? 0u : o.codes(__uint_as_float(s << 23));
      }
      __builtin_memcpy(__builtin_assume_aligned(codes + (lane * COLS + c) * PITCH + b * 16, 16), out, 16);
      scales[(lane * COLS + c) * 8 + b] = (uint8_t)s;
    }
  }
  __syncthreads();
  const int blocks = (int)(nb - b0 < 8 ? nb - b0 : 8);
#pragma unroll
  for (int i = 0; i < ROWS / 64; ++i) {
    const int row = i * 64 + tid / 8, b = tid % 8;
    if (m0 + row >= M || b >= blocks) continue;
    const i32x4 v = *(const i32x4*)(codes + row * PITCH + b * 16);
    *((i32x4*)q + (m0 + row) * nb + b0 + b) = v;
  }
  if (tid < ROWS && m0 + tid < M) {
    uint8_t* p = scale + (m0 + tid) * nb + b0;
    if (blocks == 8) {
      __builtin_memcpy(p, __builtin_assume_aligned(scales + tid * 8, 8), 8);
    } else {
      for (int b = 0; b < blocks; ++b) p[b] = scales[tid * 8 + b];
    }
  }
}

// The inverse, rounded once to the output's type: v_cvt_scalef32_pk_*_fp4, which gives NaN for s = 255. A lane makes
// 16 bytes, 8 values of 16 bits or 4 of 32, so that a wave's store is one run. STREAM: stores that leave the caches
// alone, for rows of whole 16 bytes (8192x8192 to fp32: 42 against 64 us, 16384x16384 to bf16: 93 and 126, 2048x4096:
// 3.8 and 4.7); with others they meet cache lines in parts (5000x8001 to fp32: 35 against 31 us).
template <int TYPE, bool STREAM>
__global__ void __launch_bounds__(256)
dequantize_kernel(const void* __restrict__ qv, const uint8_t* __restrict__ scale, void* __restrict__ xv, size_t first,
                  size_t items, uint32_t row_items, int64_t K) {
  typedef typename Elem<TYPE>::bits bits;
  constexpr int V = 16 / (int)sizeof(bits);
  const size_t base = first + (size_t)blockIdx.x * 256;
  const size_t i = base + threadIdx.x;
  if (i >= items) return;
  const size_t row0 = base / row_items;
  const uint32_t at = (uint32_t)(base - row0 * row_items) + threadIdx.x, over = at / row_items;
  const int64_t k0 = (int64_t)(at - over * row_items) * V;
  const float s = __uint_as_float((uint32_t)scale[i / (32 / V)] << 23);
  u32x4_any w;
  if constexpr (TYPE == FP32) {
    const uint32_t c = ((const uint16_t*)qv)[i];
    const f32x2 v[2] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1)};
    __builtin_memcpy(&w, v, 16);
  } else if constexpr (TYPE == BF16) {
    const uint32_t c = ((const uint32_t*)qv)[i];
    const bf16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3)};
    __builtin_memcpy(&w, v, 16);
  } else {
    const uint32_t c = ((const uint32_t*)qv)[i];
    const f16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 3)};
    __builtin_memcpy(&w, v, 16);
  }
  bits* p = (bits*)xv + (int64_t)(row0 + over) * K + k0;
  if (k0 + V <= K) {
    if constexpr (STREAM) __builtin_nontemporal_store(w, (u32x4_any*)p);
    else *(u32x4_any*)p = w;
  } else {
    bits t[V];
    __builtin_memcpy(t, &w, 16);
#pragma unroll
    for (int j = 0; j < V; ++j)
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

template <typename OutT>
__global__ void __launch_bounds__(256) zero_kernel(OutT* __restrict__ C, size_t first, size_t n) {
  const size_t i = first + (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) C[i] = (OutT)0.f;
}

// Tile of workgroup w. Workgroups go to the 8 XCDs in turn; each XCD gets a run of consecutive tiles, and a run
// walks groups of GROUP tile rows down and then right, so that what is in an XCD's L2 is used by its neighbours.
// Groups start at columns of their own: where all start at the first, the XCDs ask HBM for the same rows of B at
// one time, in every round of tiles again (8192^3, codes not yet in the Infinity cache: 267 against 253 us).
__device__ __forceinline__ void tile_of(uint32_t w, int tiles_m, int tiles_n, int& tm, int& tn) {
  constexpr uint32_t GROUP = 4;
  const uint32_t n = (uint32_t)tiles_m * tiles_n, x = w & 7, q = n >> 3, rest = n & 7;
  const uint32_t t = x * q + min(x, rest) + (w >> 3);
  const uint32_t in_group = GROUP * tiles_n, group = t / in_group, first = group * GROUP;
  const uint32_t rows = min((uint32_t)tiles_m - first, GROUP), groups = (tiles_m + GROUP - 1) / GROUP;
  tm = (int)(first + t % in_group % rows);
  tn = (int)((t % in_group / rows + group * tiles_n / groups) % tiles_n);
}

// ---------------------------------------------------------------------------
// Large products. A workgroup of 4 waves makes a tile of C of 64 T x 64 T, each wave a quarter of T x T tiles of
// 32x32 (v_mfma_scale_f32_32x32x64_f8f6f4: lane l holds chunk l / 32 of row l % 32 and that block's scale).
// K goes by in tiles of 8 blocks (256 values, 128 B a row), STAGES of them in LDS:
//   * codes HBM -> LDS without registers (global_load_lds, 16 B a lane), 16-byte slot s of row r holding chunk
//     s ^ (r / 2 % 8), so that 16 rows' reads of one chunk meet all 64 banks once;
//   * step s = 0 .. 3 of a tile gives lane l the chunk 4 (l / 32) + s: its four scales are neighbours, one
//     32-bit word, which the instruction's byte select takes apart.
// While a step's products run, the next step's fragments are read into the other register set; the one barrier
// of a tile stands before its last step, where its last read has returned and the next tile has arrived.
// B's rows are the instruction's rows, A's its columns: a lane ends with 4 neighbours of a row of C. The sums
// go through LDS once more, so that whole cache lines are stored.
// Tiles at the lower and right edge are moved up and left into C; what two tiles cover both write alike.
template <int N, typename F, int... I>
__device__ __forceinline__ void unroll_(F f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, typename F>
__device__ __forceinline__ void unroll(F f) { unroll_<N>(f, std::make_integer_sequence<int, N>{}); }

typedef __attribute__((address_space(3))) void lds_void;

constexpr int tile_lds(int BM, int BN, int stages) { return stages * (BM + BN) * 128; }

template <int S>   // acc += a b^T with byte S of the scales
__device__ __forceinline__ void mfma32(f32x16& acc, i32x4 a, i32x4 b, uint32_t sa, uint32_t sb) {
  acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(frag(a), frag(b), acc, 4, 4, S, (int)sa, S, (int)sb);
}

constexpr int waitcnt(int vm, int lgkm) { return (vm & 15) | (vm >> 4) << 14 | 7 << 4 | lgkm << 8; }   // s_waitcnt's operand

template <typename OutT, int T, int STAGES>
__global__ void __launch_bounds__(256, 2)
gemm_tile_kernel(const uint8_t* __restrict__ A, const uint8_t* __restrict__ As, const uint8_t* __restrict__ B,
                 const uint8_t* __restrict__ Bs, OutT* __restrict__ C, int M, int N, int nb_all, int per, float alpha, int stream) {
  constexpr int BM = 64 * T, BN = 64 * T;
  constexpr int DATA = (BM + BN) * 128;
  constexpr bool DEEP = T == 1;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // STAGES x codes of A, B
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int wm = wave >> 1, wn = wave & 1;
  int tm, tn;
  const int tiles_m = (M + BM - 1) / BM;
  tile_of(blockIdx.x, tiles_m, (N + BN - 1) / BN, tm, tn);
  const int m0 = min(tm * BM, M - BM), n0 = min(tn * BN, N - BN);
  const int first = (int)blockIdx.y * per;                // this part of K: its blocks, tiles, blocks of the last tile
  const int nb = min(nb_all - first * 8, per * 8), nt = (nb + 7) / 8, rem = nb - (nt - 1) * 8;
  C += (size_t)blockIdx.y * M * N;

  // staging: a wave's load takes 8 rows of 128 B, and 32 rows on with the next
  const size_t row_bytes = (size_t)nb_all * 16;
  const int srow = wave * 8 + (lane >> 3), chunk = (lane & 7) ^ ((srow >> 1) & 7);
  const uint32_t off = (uint32_t)srow * (uint32_t)row_bytes + chunk * 16;
  const uint8_t* const tA = A + (size_t)m0 * row_bytes + (size_t)first * 128;
  const uint8_t* const tB = B + (size_t)n0 * row_bytes + (size_t)first * 128;
  constexpr int LOADS = (BM + BN) / 32;
  auto stage = [&](int t, int buffer, int j) {
    uint32_t o = off;
    if (t == nt - 1 && chunk >= rem) o -= (uint32_t)(chunk - rem + 1) * 16;   // behind the last block: that one again
    const uint8_t* p = (j < BM / 32 ? tA + j * 32 * row_bytes : tB + (j - BM / 32) * 32 * row_bytes) + (size_t)t * 128;
    __builtin_amdgcn_global_load_lds((const void*)(p + o), (lds_void*)(lds + buffer * DATA + wave * 1024 + j * 4096), 16, 0, 0);
  };

  // Scales. A row's 32 bytes of 4 tiles are read at a time, a batch ahead, lane (r, h) taking tiles 2 h and 2 h + 1; the
  // halves of the wave then swap, each keeping its half of every 8 bytes. Of a short last tile the 8 bytes that end
  // with the row are read, and moved down; where the row has fewer than 8, one by one.
  constexpr int GROUPS = 2 * T;
  struct Scales { uint32_t v[GROUPS]; } sc, queue[4];   // of A's row groups, then B's: this tile's, 4 tiles'
  uint64_t batch[GROUPS][2];
  const uint8_t* sp[GROUPS];
#pragma unroll
  for (int n = 0; n < GROUPS; ++n)
    sp[n] = (n < T ? As + (size_t)(m0 + (wm * T + n) * 32 + r) * nb_all : Bs + (size_t)(n0 + (wn * T + n - T) * 32 + r) * nb_all) + first * 8;
  auto sload = [&](int t) {
#pragma unroll
    for (int n = 0; n < GROUPS; ++n) {
      const uint8_t* p = sp[n] + (size_t)t * 8 + h * 16;
      if (t * 8 + 32 <= nb) {
        __builtin_memcpy(batch[n], p, 16);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = t + h * 2 + i;
          if (at >= nt) continue;
          if (nb < 8) {
            batch[n][i] = 0;
            for (int k = 0; k < rem; ++k) batch[n][i] |= (uint64_t)p[k] << (8 * k);
            continue;
          }
          const int back = at == nt - 1 ? 8 - rem : 0;
          __builtin_memcpy(&batch[n][i], p + i * 8 - back, 8);
          batch[n][i] >>= 8 * back;
        }
      }
    }
  };
  auto sask = [&](int t, auto u) {   // in tile t, u = t % 4, for the 4 tiles behind these
    if constexpr (u == 0)
      if (t + 4 < nt) sload(t + 4);
  };
  auto snext = [&](auto u) {   // to a tile t with u = t % 4
    if constexpr (u == 0) {
#pragma unroll
      for (int n = 0; n < GROUPS; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap((uint32_t)batch[n][i], (uint32_t)(batch[n][i] >> 32), false, false));
          queue[i].v[n] = v.x;
          queue[2 + i].v[n] = v.y;
        }
    }
    sc = queue[u];
  };

  // Fragments, by step: of a whole tile and the next one, or of a step and the next.
  const int baseA = (wm * 32 * T + r) * 128, baseB = BM * 128 + (wn * 32 * T + r) * 128;
  struct Frags { i32x4 a[T], b[T]; } f[DEEP ? 8 : 2];
  auto read_one = [&](int buffer, auto s, Frags& to, int k) {   // b0 a0 b1 a1 ..
    const uint8_t* p = lds + buffer * DATA + (((4 * h + s) ^ ((r >> 1) & 7)) << 4);
    if (k % 2 == 0) to.b[k / 2] = *(const i32x4*)(p + baseB + k / 2 * 4096);
    else to.a[k / 2] = *(const i32x4*)(p + baseA + k / 2 * 4096);
  };
  // Of step s, two at a time, asked for in the first groups of the step before: the last of them is on its way while
  // the other groups' products run.
  auto read = [&](int buffer, auto s, int pair) {
    if (2 * pair >= GROUPS) return;
    read_one(buffer, s, f[s % 2], 2 * pair);
    read_one(buffer, s, f[s % 2], 2 * pair + 1);
  };

  f32x16 acc[T][T];
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  // Step s on one register set, in groups: some of the products, then ask(k) asks for something. Asked for before
  // the first product, it would be in what that product waits for.
  auto step = [&](auto s, auto ask) {
    unroll<GROUPS>([&](auto k) {
      unroll<T * T>([&](auto p) {
        if constexpr (p * GROUPS / (T * T) == k)
          mfma32<s>(acc[p / T][p % T], f[s % 2].b[p % T], f[s % 2].a[p / T], sc.v[T + p % T], sc.v[p / T]);
      });
      __builtin_amdgcn_sched_barrier(0);
      ask(k);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // All but the last KEEP loads that this wave asked for are in LDS, what it read is in registers; then everyone's.
  auto landed = [](auto keep) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(waitcnt(keep, 0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::integral_constant<int, 0> s0{};
  constexpr std::integral_constant<int, 1> s1{};
  constexpr std::integral_constant<int, 2> s2{};
  constexpr std::integral_constant<int, 3> s3{};
  constexpr std::false_type no{};
  constexpr std::true_type yes{};
  static_assert(LOADS == 2 * GROUPS, "a load for each group of two steps");

  // Tile t in buffer u % STAGES, u = t % 4. The loads of a tile are spread over the last step of the tile STAGES
  // before it and the first of the next one: they pass the vector memory pipe at 16 cycles each for the whole
  // workgroup. full: all tiles that it asks for are there; else it sees which are, and whether it is the last.
  auto tile = [&](int t, auto u, auto full) {
    constexpr int HERE = u % STAGES, NEXT = (u + 1) % STAGES, BEFORE = (u + STAGES - 1) % STAGES;
    const bool next = full || t + 1 < nt;
    auto clear = [&](auto s) {   // what is behind the last block is multiplied by zeros
      if (!full && !next && 4 * h + s >= rem) {
#pragma unroll
        for (int i = 0; i < T; ++i) f[s % 2].a[i] = i32x4{0, 0, 0, 0};
      }
    };
    clear(s0);
    step(s0, [&](auto k) {
      read(HERE, s1, k);
      if (full || t + STAGES - 1 < nt) stage(t + STAGES - 1, BEFORE, LOADS / 2 + k);
      if constexpr (k == 0) sask(t, u);
    });
    clear(s1);
    step(s1, [&](auto k) { read(HERE, s2, k); });
    clear(s2);
    step(s2, [&](auto k) { read(HERE, s3, k); });
    if (full) {
      landed(std::integral_constant<int, (STAGES - 2) * LOADS>{});
    } else if (STAGES > 2 && t + 3 < nt) {
      landed(std::integral_constant<int, STAGES == 4 ? 2 * LOADS : 0>{});
    } else if (STAGES > 2 && t + 2 < nt) {
      landed(std::integral_constant<int, STAGES == 4 ? LOADS : 0>{});
    } else {
      landed(s0);
    }
    clear(s3);
    step(s3, [&](auto k) {
      if (next) read(NEXT, s0, k);
      if (full || t + STAGES < nt) stage(t + STAGES, HERE, k);
    });
    if (next) snext(std::integral_constant<int, (u + 1) % 4>{});
    return next;
  };
  static_assert(STAGES == 2 || STAGES == 4, "a buffer follows from t % 4");

  // The same for T = 1, whose step has less to multiply than an LDS read takes: it reads the next tile's fragments of
  // all steps behind the products of its first, and asks for the tile STAGES on behind the second's (2048x1024x4096 to
  // bf16: 9.3 against 9.8 us, 128x4096x4096: 6.1 and 7.0; for T = 2 it is slower, 12.8 and 11.3).
  auto deep = [&](int t, auto u, auto full) {
    constexpr int HERE = u % STAGES, NEXT = (u + 1) % STAGES;
    Frags* const here = f + (u % 2) * 4;
    Frags* const ahead = f + ((u + 1) % 2) * 4;
    const bool next = full || t + 1 < nt;
    if (full) {
      landed(std::integral_constant<int, (STAGES - 2) * LOADS>{});
    } else if (STAGES > 2 && t + 3 < nt) {
      landed(std::integral_constant<int, STAGES == 4 ? 2 * LOADS : 0>{});
    } else if (STAGES > 2 && t + 2 < nt) {
      landed(std::integral_constant<int, STAGES == 4 ? LOADS : 0>{});
    } else {
      landed(s0);
    }
    unroll<4>([&](auto s) {
      if (!full && !next && 4 * h + s >= rem) {
#pragma unroll
        for (int i = 0; i < T; ++i) here[s].a[i] = i32x4{0, 0, 0, 0};
      }
      unroll<T * T>([&](auto p) {
        mfma32<s>(acc[p / T][p % T], here[s].b[p % T], here[s].a[p / T], sc.v[T + p % T], sc.v[p / T]);
      });
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (s == 0) {
        if (next)
          unroll<4>([&](auto v) {
#pragma unroll
            for (int k = 0; k < GROUPS; ++k) read_one(NEXT, v, ahead[v], k);
          });
      }
      if constexpr (s == 1) {
        sask(t, u);
        if (full || t + STAGES < nt) {
#pragma unroll
          for (int j = 0; j < LOADS; ++j) stage(t + STAGES, HERE, j);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    if (next) snext(std::integral_constant<int, (u + 1) % 4>{});
    return next;
  };

  sload(0);
#pragma unroll
  for (int j = 0; j < LOADS; ++j) stage(0, 0, j);
  // The scales have come. Said outside of any branch: on a path that it took for possible the compiler saw them on
  // their way into the loop, and waited there for all loads, every time.
  __builtin_amdgcn_s_waitcnt(waitcnt(LOADS, 15));
  snext(s0);
#pragma unroll
  for (int i = 1; i < STAGES; ++i)
#pragma unroll
    for (int j = 0; j < (DEEP || i < STAGES - 1 ? LOADS : LOADS / 2); ++j)
      if (i < nt) stage(i, i, j);
  if (nt >= STAGES) landed(std::integral_constant<int, (STAGES - 2) * LOADS + (DEEP ? LOADS : LOADS / 2)>{});
  else landed(s0);
  if constexpr (DEEP) {
    unroll<4>([&](auto v) {
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) read_one(0, v, f[v], k);
    });
  } else {
    unroll<GROUPS>([&](auto k) { read(0, s0, k); });
  }
  auto either = [&](int t, auto u, auto full) {
    if constexpr (DEEP) return deep(t, u, full);
    else return tile(t, u, full);
  };
  int t = 0;
  for (; t + 3 + STAGES < nt; t += 4) {
    either(t, s0, yes);
    either(t + 1, s1, yes);
    either(t + 2, s2, yes);
    either(t + 3, s3, yes);
  }
  for (;;) {
    if (!either(t++, s0, no)) break;
    if (!either(t++, s1, no)) break;
    if (!either(t++, s2, no)) break;
    if (!either(t++, s3, no)) break;
  }
  landed(s0);   // no wave reads codes any more

  // Element e of lane (r, h) of a 32x32 tile: column r, row 8 (e / 4) + 4 h + e % 4. 32 rows of C go through the
  // wave's part of LDS at a time, 16 bytes apart from a multiple of the banks.
  constexpr int ROW = 32 * T * (int)sizeof(OutT), PITCH = ROW + 16;
  constexpr int LANES = ROW / 16, ROWS = 64 / LANES;   // of a store
  static_assert(32 * PITCH <= tile_lds(BM, BN, STAGES) / 4, "a wave's part of LDS");
  uint8_t* const mine = lds + wave * (tile_lds(BM, BN, STAGES) / 4);
#pragma unroll
  for (int i = 0; i < T; ++i) {
#pragma unroll
    for (int j = 0; j < T; ++j) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        OutT v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (OutT)(alpha * acc[i][j][q * 4 + e]);
        __builtin_memcpy(__builtin_assume_aligned(mine + r * PITCH + (j * 32 + q * 8 + h * 4) * sizeof(OutT), sizeof v), v, sizeof v);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint8_t* p = (uint8_t*)(C + (size_t)(m0 + (wm * T + i) * 32) * N + n0 + wn * 32 * T);
#pragma unroll
    for (int k = 0; k < 32 / ROWS; ++k) {
      const int row = k * ROWS + lane / LANES, at = lane % LANES * 16;
      const i32x4 v = *(const i32x4*)(mine + row * PITCH + at);
      u32x4_any* to = (u32x4_any*)(p + (size_t)row * N * sizeof(OutT) + at);
      if (stream) __builtin_nontemporal_store(__builtin_bit_cast(u32x4_any, v), to);
      else *to = __builtin_bit_cast(u32x4_any, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// ---------------------------------------------------------------------------
// The largest products: tiles of 256x256 on v_mfma_scale_f32_16x16x128_f8f6f4, a wave having 8x8 of 16x16. The same
// staging of K, with two steps a tile: step s = 0, 1 gives lane (r, g) = (l % 16, l / 16) the chunk 2 g + s. A CU holds
// one workgroup, a SIMD one wave, with all 512 registers: 256 of sums, two sets of fragments.
// At full rate this runs into the card's power, so that what counts is energy: products alone, from registers, of
// random codes, run at 7.2 PFLOP/s in this form and 6.5 as 32x32x64 (8.3 both, of zeros). 8192^3 takes 252 us to fp32
// and 232 to bf16 with the scales' launch, 4.4 and 4.7 PFLOP/s, at 1.85 of 2.4 GHz, products in 62 % of the cycles; about
// half of the rest is the write of C at the end of each of 4 rounds, by all CUs at one time (11 us a round to fp32).

// Scales in the order in which the lanes take them: panel (a wave's 128 rows) by tile of K, 64 lanes of 16 bytes, lane
// (r, g) having the 16 bits of its chunks 2 g and 2 g + 1 of rows r, 16 + r, .. 112 + r. Read where they lie, a row's 8
// bytes a tile cost a cache line each; at 8192^3 that made the product 11 % slower than this kernel and its launch do.
// A workgroup turns 8 tiles of a panel, 64 bytes a row, over in LDS. Blocks behind the last read as 0, which
// multiplies zeros.
__global__ void __launch_bounds__(256)
arrange_scales_kernel(const uint8_t* __restrict__ As, const uint8_t* __restrict__ Bs, uint8_t* __restrict__ out, int M, int N,
                      int nb) {
  constexpr int PITCH = 68;   // 17 banks: 16 rows' words of one tile lie in different ones
  __shared__ __attribute__((aligned(16))) uint8_t rows[128 * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int nt = (nb + 7) / 8, t0 = (int)blockIdx.y * 8;
  const int panels_a = (M + 255) / 256 * 2, panel = (int)blockIdx.x;
  const bool isA = panel < panels_a;
  const int q = isA ? panel : panel - panels_a, all = isA ? M : N;
  const int row0 = min(q / 2 * 256, all - 256) + q % 2 * 128;
  const uint8_t* s = isA ? As : Bs;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = i * 64 + tid / 4, c = t0 * 8 + tid % 4 * 16;
    const uint8_t* p = s + (size_t)(row0 + row) * nb + c;
    uint32_t v[4] = {0, 0, 0, 0};
    if (c + 16 <= nb) {
      __builtin_memcpy(v, p, 16);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (c + k < nb) v[k / 4] |= (uint32_t)p[k] << (8 * (k % 4));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) *(uint32_t*)(rows + row * PITCH + tid % 4 * 16 + k * 4) = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = i * 4 + tid / 64;
    if (t0 + t >= nt) continue;
    uint16_t v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = *(const uint16_t*)(rows + (k * 16 + r) * PITCH + t * 8 + g * 2);
    __builtin_memcpy(__builtin_assume_aligned(out + (((size_t)panel * nt + t0 + t) * 64 + lane) * 16, 16), v, 16);
  }
}

// acc += a b^T with byte SA, SB of the scales, in place in the accumulation registers. The compiler's own form gives
// the sum another place and moves it back, which with 256 of them costs more than the products. What inline assembly
// has to see to: 2 wait states between an ordinary instruction's write of an operand and this one, which the callers
// keep (with an s_nop before each the kernel is 3 % slower; a test looks for it in the assembly), and the wait before a
// sum is read, which is settle's. Sums are used again 64 instructions later, after any wait there is.
template <int SA, int SB>
__device__ __forceinline__ void mfma16(f32x4& acc, i32x4 a, i32x4 b, uint32_t sa, uint32_t sb) {
  asm volatile(
      "v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
      : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb), "i"(SA & 1), "i"(SB & 1), "i"(SA >> 1), "i"(SB >> 1));
}
// Once all are waited for, each sum is bound behind that wait.
__device__ __forceinline__ void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }
__device__ __forceinline__ void settled(f32x4& acc) { asm volatile("" : "+a"(acc)); }

// Slot s of row r holds chunk s ^ turn(r) here. A quarter of a wave's reads is not 16 lanes in a row: with rows 0 .. 3
// and 12 .. 15 of one chunk go rows 4 .. 11 of the chunk 2 on, and s ^ (r / 2 % 8) has them meet in half the banks.
__device__ __forceinline__ int turn(int row) { return ((row >> 1) & 7) ^ (row & 4); }

// S: what arrange_scales_kernel left, of both operands
template <typename OutT>
__global__ void __launch_bounds__(256, 1)
gemm_large_kernel(const uint8_t* __restrict__ A, const uint8_t* __restrict__ B, const uint8_t* __restrict__ S,
                  OutT* __restrict__ C, int M, int N, int nb, float alpha, int stream) {
  constexpr int B0 = 256 * 128, DATA = 2 * B0, LOADS = 16;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // 2 x codes of A, B
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int wm = wave >> 1, wn = wave & 1;
  int tm, tn;
  const int tiles_m = (M + 255) / 256;
  tile_of(blockIdx.x, tiles_m, (N + 255) / 256, tm, tn);
  const int m0 = min(tm * 256, M - 256), n0 = min(tn * 256, N - 256);
  const int nt = (nb + 7) / 8, rem = nb - (nt - 1) * 8;   // tiles of K, blocks of the last

  // staging: a wave's load takes 8 rows of 128 B, and 32 rows on with the next; inner: not of the last tile
  const size_t row_bytes = (size_t)nb * 16;
  const int srow = wave * 8 + (lane >> 3), chunk = (lane & 7) ^ turn(srow);
  const uint32_t off = (uint32_t)srow * (uint32_t)row_bytes + chunk * 16;
  const uint8_t* const tA = A + (size_t)m0 * row_bytes;
  const uint8_t* const tB = B + (size_t)n0 * row_bytes;
  auto stage = [&](int t, int buffer, int j, bool inner) {
    uint32_t o = off;
    if (!inner && t == nt - 1 && chunk >= rem) o -= (uint32_t)(chunk - rem + 1) * 16;   // behind the last block: that one again
    const uint8_t* p = (j < 8 ? tA + j * 32 * row_bytes : tB + (j - 8) * 32 * row_bytes) + (size_t)t * 128;
    __builtin_amdgcn_global_load_lds((const void*)(p + o), (lds_void*)(lds + buffer * DATA + wave * 1024 + j * 4096), 16, 0, 0);
  };

  // scales of A's 8 row groups and B's, 16 bits each: this tile's and the next's
  struct Scales { uint32_t a[4], b[4]; } sc, sn;
  const uint8_t* const sA = S + (size_t)(tm * 2 + wm) * nt * 1024 + lane * 16;
  const uint8_t* const sB = S + (size_t)((tiles_m + tn) * 2 + wn) * nt * 1024 + lane * 16;
  auto sload = [&](int t) {
    __builtin_memcpy(sn.a, __builtin_assume_aligned(sA + (size_t)t * 1024, 16), 16);
    __builtin_memcpy(sn.b, __builtin_assume_aligned(sB + (size_t)t * 1024, 16), 16);
  };

  // fragments of a step and the next; 0 .. 7 are B's, 8 .. 15 A's
  struct Frags { i32x4 b[8], a[8]; } f[2];
  const int base = r * 128, at[2] = {((2 * g) ^ turn(r)) << 4, ((2 * g + 1) ^ turn(r)) << 4};
  auto read = [&](int buffer, auto s, int k) {
    const uint8_t* p = lds + buffer * DATA + base + at[s];
    if (k % 2 == 0) f[s].b[k / 2] = *(const i32x4*)(p + B0 + (wn * 8 + k / 2) * 2048);
    else f[s].a[k / 2] = *(const i32x4*)(p + (wm * 8 + k / 2) * 2048);
  };

  f32x4 acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Step s on one set: 64 products, and behind product p ask(p) asks for something. Asked for before the first product,
  // it would be in what that product waits for. From one product to the next one operand stays, also where a row of
  // them ends (8192^3: 256.3 -> 254.3 us, for what the change of an operand costs in power).
  auto step = [&](auto s, auto ask) {
    unroll<64>([&](auto p) {
      constexpr int i = p / 8, j = i % 2 ? 7 - p % 8 : p % 8;
      mfma16<j % 2 * 2 + s, i % 2 * 2 + s>(acc[i][j], f[s].b[j], f[s].a[i], sc.b[j / 2], sc.a[i / 2]);
      __builtin_amdgcn_sched_barrier(0);
      ask(p);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto landed = [](auto keep) {   // as above
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(waitcnt(keep, 0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  auto wait_states = [] {   // between ordinary instructions before and products behind
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 1");
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::integral_constant<int, 0> s0{};
  constexpr std::integral_constant<int, 1> s1{};
  constexpr std::false_type no{};
  constexpr std::true_type yes{};

  // Tile t in buffer u = t % 2. The loads of a tile are spread over the second step of the tile two before it: they
  // pass the vector memory pipe at 16 cycles each for the whole workgroup. Half of them a step later, when HBM has
  // less than a step to answer, and 8192^3 takes 7 % longer. full: it asks for no tile that is not there, nor for the
  // last.
  auto tile = [&](int t, auto u, auto full) {
    const bool next = full || t + 1 < nt;
    auto clear = [&](auto s) {   // what is behind the last block is multiplied by zeros
      if (!full && !next && 2 * g + s >= rem) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[s].a[i] = i32x4{0, 0, 0, 0};
      }
      if (!full) wait_states();
    };
    clear(s0);
    step(s0, [&](auto p) {
      if constexpr (p % 2 == 0 && p / 2 < 16) read(u, s1, p / 2);
      if constexpr (p == 3)
        if (next) sload(t + 1);
    });
    landed(s0);
    clear(s1);
    step(s1, [&](auto p) {
      if constexpr (p % 2 == 0 && p / 2 < 16)
        if (next) read(1 - u, s0, p / 2);
      if constexpr (p % 4 == 1)
        if (full || t + 2 < nt) stage(t + 2, u, p / 4, full);
    });
    if (next) {
      sc = sn;
      wait_states();
    }
    return next;
  };

  sload(0);
#pragma unroll
  for (int j = 0; j < LOADS; ++j) stage(0, 0, j, false);
  __builtin_amdgcn_s_waitcnt(waitcnt(LOADS, 15));   // the scales have come, outside of any branch, as above
  sc = sn;
  if (nt > 1) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) stage(1, 1, j, false);
    landed(std::integral_constant<int, LOADS>{});
  } else {
    landed(s0);
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) read(0, s0, k);
  int t = 0;
  for (; t + 4 < nt; t += 2) {
    tile(t, s0, yes);
    tile(t + 1, s1, yes);
  }
  for (;;) {
    if (!tile(t++, s0, no)) break;
    if (!tile(t++, s1, no)) break;
  }
  landed(s0);   // no wave reads codes any more
  settle();

  // element e of lane (r, g) of a 16x16 tile: column r, row 4 g + e. 32 rows of C at a time, as above
  constexpr int ROW = 128 * (int)sizeof(OutT), PITCH = ROW + 16;
  constexpr int LANES = ROW / 16, ROWS = 64 / LANES;
  static_assert(32 * PITCH <= DATA / 2, "a wave's part of LDS");
  uint8_t* const mine = lds + wave * (DATA / 2);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        settled(acc[i + h][j]);
        OutT v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (OutT)(alpha * acc[i + h][j][e]);
        __builtin_memcpy(__builtin_assume_aligned(mine + (h * 16 + r) * PITCH + (j * 16 + g * 4) * sizeof(OutT), sizeof v), v, sizeof v);
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint8_t* p = (uint8_t*)(C + (size_t)(m0 + wm * 128 + i * 16) * N + n0 + wn * 128);
#pragma unroll
    for (int k = 0; k < 32 / ROWS; ++k) {
      const int row = k * ROWS + lane / LANES, to = lane % LANES * 16;
      const u32x4_any v = __builtin_bit_cast(u32x4_any, *(const i32x4*)(mine + row * PITCH + to));
      u32x4_any* out = (u32x4_any*)(p + (size_t)row * N * sizeof(OutT) + to);
      if (stream) __builtin_nontemporal_store(v, out);
      else *out = v;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// Products of few rows, whose time is the reading of the other operand. P is the operand with the many rows, Q that
// with the few; a workgroup makes NP x NQ tiles of 16x16 (v_mfma_scale_f32_16x16x128_f8f6f4), its WAVES taking units
// of 8 blocks (256 values, 128 B a row) of K in turn, each through two buffers of its own in LDS: no wave waits for
// another before the sums meet, in the order of the waves. (Straight to registers the instruction's layout has
// neighbouring lanes read different rows, 16 bytes of each: 32x8192x8192 took 13.3 us so.) With four waves the compiler
// gives registers of the scales to addresses, and waits for all loads on their way before it asks for a wave's next unit:
// the second buffer hides little there. Slots in LDS are those of the largest tile, and what is read behind the last row
// and block is as there; lane (r, g) takes chunks 2 g and 2 g + 1 of row r, whose scales are one 16-bit word, the
// instruction's byte select taking them apart.
constexpr int rows_lds(int NP, int NQ, int WAVES) { return WAVES * 2 * (NP + NQ) * 16 * 128; }

template <typename OutT, int NP, int NQ, int WAVES>
__global__ void __launch_bounds__(WAVES * 64)
gemm_rows_kernel(const uint8_t* __restrict__ P, const uint8_t* __restrict__ Ps, const uint8_t* __restrict__ Q,
                 const uint8_t* __restrict__ Qs, OutT* __restrict__ C, int np, int nq, int nb_all, int per, int64_t cp,
                 int64_t cq, float alpha) {
  constexpr int GROUPS = NP + NQ, UNIT = GROUPS * 16 * 128, LOADS = GROUPS * 2;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int tiles_p = (np + NP * 16 - 1) / (NP * 16);
  const int p0 = (int)(blockIdx.x % tiles_p) * NP * 16, q0 = (int)(blockIdx.x / tiles_p) * NQ * 16;
  const int first = (int)blockIdx.y * per;   // this part of K: its blocks, whole units, blocks of a short one
  const int nb = min(nb_all - first * 8, per * 8), units = nb / 8, rem = nb % 8;
  C += (size_t)blockIdx.y * np * nq;
  uint8_t* const mine = lds + wave * 2 * UNIT;

  // the block that row i starts with of the 16 GROUPS
  auto row = [&](int i) { return (size_t)(i < NP * 16 ? min(p0 + i, np - 1) : min(q0 + i - NP * 16, nq - 1)) * nb_all + (size_t)first * 8; };
  size_t from[LOADS];   // a load takes 8 rows of 128 B
  const int chunk[2] = {(lane & 7) ^ turn(lane >> 3), (lane & 7) ^ turn(8 + (lane >> 3))};   // of even loads, of odd ones
#pragma unroll
  for (int j = 0; j < LOADS; ++j) from[j] = (row(j * 8 + (lane >> 3)) + chunk[j % 2]) * 16;
  size_t srow[GROUPS];
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) srow[i] = row(i * 16 + r);

  struct Scales { uint32_t v[GROUPS]; };
  auto load = [&](int t, int buffer, Scales& s, auto part) {
    // The buffer's last reads have returned. Its products, which are behind them, wait for that too, but nothing keeps the
    // compiler from moving those behind these loads.
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(waitcnt(63, 0));
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      const uint8_t* p = (i < NP ? Ps : Qs) + srow[i] + (size_t)t * 8 + g * 2;
      if (part) {   // 1 behind the last block
        s.v[i] = (g * 2 < rem ? p[0] : 127) | (g * 2 + 1 < rem ? p[1] : 127) << 8;
      } else {
        uint16_t v;
        __builtin_memcpy(&v, p, 2);
        s.v[i] = v;
      }
    }
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const uint8_t* p = (j < NP * 2 ? P : Q) + from[j] + (size_t)t * 128;
      if (part && chunk[j % 2] >= rem) p -= (chunk[j % 2] - rem + 1) * 16;
      __builtin_amdgcn_global_load_lds((const void*)p, (lds_void*)(mine + buffer * UNIT + j * 1024), 16, 0, 0);
    }
  };
  f32x4 acc[NP][NQ];
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int j = 0; j < NQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int buffer, const Scales& s, auto part) {
    unroll<2>([&](auto k) {
      i32x4 v[GROUPS];
#pragma unroll
      for (int i = 0; i < GROUPS; ++i)
        v[i] = *(const i32x4*)(mine + buffer * UNIT + (i * 16 + r) * 128 + (((2 * g + k) ^ turn(r)) << 4));
      if (part && 2 * g + k >= rem) {
#pragma unroll
        for (int j = 0; j < NQ; ++j) v[NP + j] = i32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(frag(v[i]), frag(v[NP + j]), acc[i][j], 4, 4, k,
                                                                        (int)s.v[i], k, (int)s.v[NP + j]);
    });
  };
  auto arrived = [](auto keep) {   // all but the last of this wave's loads
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(waitcnt(keep, 15));
    asm volatile("" ::: "memory");
  };
  constexpr std::integral_constant<int, 0> none{};
  constexpr std::false_type whole{};
  constexpr std::true_type part{};
  // unit t in one buffer, the wave's next on its way into the other
  Scales s[2];
  auto unit = [&](int t, auto buffer) {
    const bool more = t + WAVES < units;
    if (more) {
      load(t + WAVES, 1 - buffer, s[1 - buffer], whole);
      arrived(std::integral_constant<int, LOADS>{});
      multiply(buffer, s[buffer], whole);
    } else {
      arrived(none);
      multiply(buffer, s[buffer], whole);
    }
    return more;
  };
  int t = wave;
  if (t < units) {
    load(t, 0, s[0], whole);
    for (;; t += 2 * WAVES) {
      if (!unit(t, none)) break;
      if (!unit(t + WAVES, std::integral_constant<int, 1>{})) break;
    }
  }
  if (rem && wave == units % WAVES) {
    load(units, 0, s[0], part);
    arrived(none);
    multiply(0, s[0], part);
  }
  __syncthreads();
  f32x4* const sums = (f32x4*)lds;   // [WAVES][NP * NQ][64]
  static_assert(WAVES * NP * NQ * 1024 <= rows_lds(NP, NQ, WAVES), "the sums' place");
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int j = 0; j < NQ; ++j) sums[(wave * NP * NQ + i * NQ + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int k = wave; k < NP * NQ; k += WAVES) {
    f32x4 sum = sums[k * 64 + lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += sums[(w * NP * NQ + k) * 64 + lane];
    const int p = p0 + k / NQ * 16 + g * 4, q = q0 + k % NQ * 16 + r;
    if (q >= nq) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (p + e < np) store_out(C + (p + e) * cp + q * cq, alpha * sum[e]);
  }
}

// The sum of the parts of K, in their order. A part is 4 MiB at most and has just been written: a few microseconds.
template <typename OutT>
__global__ void __launch_bounds__(256)
join_kernel(const float* __restrict__ parts, OutT* __restrict__ C, size_t n, int count, float alpha) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float sum = parts[i];
  for (int k = 1; k < count; ++k) sum += parts[k * n + i];
  store_out(C + i, alpha * sum);
}

// bf16 values, uniform in [-1, 1), by their index: the burn-in's operands
__global__ void __launch_bounds__(256) fill_kernel(uint16_t* __restrict__ x, size_t n) {
  const size_t stride = (size_t)gridDim.x * 256;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
    uint32_t h = (uint32_t)i * 2654435761u ^ (uint32_t)(i >> 32);
    h ^= h >> 15;
    h *= 0x2c1b3c6du;
    h ^= h >> 13;
    x[i] = __builtin_bit_cast(uint16_t, (__bf16)((float)(h & 0xffffff) / 8388608.f - 1.f));
  }
}

// A launch's lanes stay below 2^32; longer runs take several launches.
constexpr size_t SLICE = (size_t)1 << 31;
// An item's place in its row has 32 bits in the kernels. A longer row is taken in pieces of this many values; its codes, its
// scales and what they stand for are one run each. No memory holds the codes of a row of LONGEST.
constexpr int64_t ROW_ITEMS = (int64_t)1 << 31, PIECE = (int64_t)1 << 32, LONGEST = (int64_t)1 << 39;

template <typename F>
static int pieces(int64_t rows, int64_t K, F launch) {
  for (int64_t r = 0; r < rows; ++r)
    for (int64_t k = 0; k < K; k += PIECE)
      if (launch(r, k, K - k < PIECE ? K - k : PIECE) != 0) return -1;
  return 0;
}

template <typename F>
static int sliced(size_t items, F launch) {
  for (size_t first = 0; first < items; first += SLICE) {
    const size_t n = items - first < SLICE ? items - first : SLICE;
    launch(first, dim3((unsigned)((n + 255) / 256)));
    HC(hipGetLastError());
  }
  return 0;
}

// The size of the tiles, in rows and columns: 0 for the small kernel, which takes everything. A round of 256 tiles,
// one for each CU, takes about 5 and 13 us at K = 4096 for tiles of 64 and 128, and 28 to 42 for 256, whose full rounds
// run into the power limit (2048x1024: 10.6 against 12.4 us; 2048x2048: 17.5 and 12.7; 4096x2560: 48, 38 and 34;
// 4096x4096: 74, 51 and 42). The proportions hold for other K but for short ones, where all store more than they
// multiply and 128 and 256 are within a fifth of each other (4096x4096x1024: 21.7 and 23.3 us to fp32;
// 8192x8192x512: 61 and 65, to bf16 53 and 43). Here and below the CUs are those of the whole card; on a partition of it,
// which has fewer, the same kernels run and none of this was measured.
static int tile_size(int64_t M, int64_t N, int64_t nb) {
  const int64_t least = M < N ? M : N;
  if (least < 64 || nb > 1 << 20) return 0;   // whole tiles inside C, 32-bit offsets in a tile
  auto rounds = [&](int64_t b) { return (((M + b - 1) / b) * ((N + b - 1) / b) + 255) / 256; };
  int best = 64;
  int64_t cost = rounds(64) * 5;
  if (least >= 128 && rounds(128) * 13 < cost) best = 128, cost = rounds(128) * 13;
  const int64_t tiles256 = ((M + 255) / 256) * ((N + 255) / 256);
  if (least >= 256 && rounds(256) * 28 + tiles256 * 14 / 256 < cost) best = 256;
  return best;
}

// K in parts, each to workgroups of its own, where a long K falls to half the CUs or fewer; join_kernel adds the sums.
// A workgroup takes about 0.22 us for a tile of K where its tiles pass through it one by one or its waves are four, and
// 0.07 with eight waves; the second launch costs 4 us, and the host 5. From 64 and 256 tiles on, in parts of 16 and 32
// or more: 64x64x16384 14.2 -> 8.3 us, 512x512x65536 83 -> 29, 1x512x65536 23 -> 9; half as long, and nothing is left
// of the gain (64x64x8192 8.5 and 7.7 us, 1x512x32768 9.5 and 7.7).
struct Split { int count, per; };   // parts, tiles of K in each
static Split split_k(int64_t M, int64_t N, int64_t nb) {
  const int64_t nt = (nb + 7) / 8, tile = tile_size(M, N, nb);
  const int64_t most = M < N ? N : M, each = ((M < N ? M : N) + 15) / 16;
  const int64_t groups = tile == 64  ? ((M + 63) / 64) * ((N + 63) / 64)
                         : tile == 0 ? (most + 15) / 16 * (each <= 2 ? 1 : (each + 3) / 4)
                                     : 256;
  const bool eight = tile == 0 && each <= 2;   // as launch_rows takes them
  if (groups > 128 || nt < (eight ? 256 : 64)) return {1, (int)nt};
  const int64_t least = eight ? 32 : 16, count = 256 / groups < nt / least ? 256 / groups : nt / least;
  const int64_t per = (nt + count - 1) / count;
  return {(int)((nt + per - 1) / per), (int)per};
}

static int64_t arranged_bytes(int64_t M, int64_t N, int64_t nb) {
  return ((M + 255) / 256 + (N + 255) / 256) * 2 * ((nb + 7) / 8) * 1024;
}

// More than 64 KiB of LDS has to be asked for, once on every device that the kernel runs on.
template <typename F>
static int allow_lds(F kernel, int bytes, std::atomic<uint64_t>& asked) {
  if (bytes <= 64 * 1024) return 0;
  int dev = 0;
  HC(hipGetDevice(&dev));
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if (bit && (asked.load(std::memory_order_relaxed) & bit)) return 0;
  HC(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  asked.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

// C past the caches, where its rows are whole 16 bytes: 2048x1024x4096 10.8 against 11.5 us, 8192x8192x2048 to bf16 94
// and 102; not a large one of a short K (8192x8192x1024 to fp32: 92 against 82 us).
static bool past_caches(const void* C, int64_t M, size_t row_bytes, int64_t nb) {
  return row_bytes % 16 == 0 && ((uintptr_t)C & 15) == 0 && (row_bytes * M <= (size_t)160 << 20 || nb >= 128);
}

template <typename OutT, int T, int STAGES>
static int launch_tile(const void* A, const void* As, const void* B, const void* Bs, void* C, int64_t M, int64_t N,
                       int64_t nb, float alpha, Split split, hipStream_t stream) {
  constexpr int BM = 64 * T, LDS = tile_lds(BM, BM, STAGES);
  if (M < BM || N < BM || nb < 1 || nb > 1 << 20)   // what the kernel's addresses assume
    return kamd_fail("gemm_mxfp4_nt: no tile of %d in %lld x %lld x %lld blocks", BM, (long long)M, (long long)N, (long long)nb);
  const int64_t tiles = ((M + BM - 1) / BM) * ((N + BM - 1) / BM);
  if (tiles >= (int64_t)1 << 24) return kamd_fail("gemm_mxfp4_nt: %lld x %lld is too large", (long long)M, (long long)N);
  auto kernel = gemm_tile_kernel<OutT, T, STAGES>;
  static std::atomic<uint64_t> asked{0};
  if (allow_lds(kernel, LDS, asked) != 0) return -1;
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, split.count), dim3(256), LDS, stream, (const uint8_t*)A, (const uint8_t*)As,
                     (const uint8_t*)B, (const uint8_t*)Bs, (OutT*)C, (int)M, (int)N, (int)nb, split.per, alpha,
                     (int)(split.count == 1 && past_caches(C, M, N * sizeof(OutT), nb)));
  return kamd_check(hipGetLastError(), "gemm_mxfp4_nt launch");
}

template <typename OutT>
static int launch_large(const void* A, const void* As, const void* B, const void* Bs, void* C, int64_t M, int64_t N,
                        int64_t nb, float alpha, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  constexpr int LDS = tile_lds(256, 256, 2);
  if (M < 256 || N < 256 || nb < 1 || nb > 1 << 20)
    return kamd_fail("gemm_mxfp4_nt: no tile of 256 in %lld x %lld x %lld blocks", (long long)M, (long long)N, (long long)nb);
  const int64_t tiles_m = (M + 255) / 256, tiles_n = (N + 255) / 256, need = arranged_bytes(M, N, nb);
  if (tiles_m * tiles_n >= (int64_t)1 << 24) return kamd_fail("gemm_mxfp4_nt: %lld x %lld is too large", (long long)M, (long long)N);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))
    return kamd_fail("gemm_mxfp4_nt: needs a workspace of %lld bytes, 16-byte aligned", (long long)need);
  auto kernel = gemm_large_kernel<OutT>;
  static std::atomic<uint64_t> asked{0};
  if (allow_lds(kernel, LDS, asked) != 0) return -1;
  hipLaunchKernelGGL(arrange_scales_kernel, dim3((unsigned)((tiles_m + tiles_n) * 2), (unsigned)((nb + 63) / 64)), dim3(256), 0,
                     stream, (const uint8_t*)As, (const uint8_t*)Bs, (uint8_t*)workspace, (int)M, (int)N, (int)nb);
  HC(hipGetLastError());
  hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles_m * tiles_n)), dim3(256), LDS, stream, (const uint8_t*)A, (const uint8_t*)B,
                     (const uint8_t*)workspace, (OutT*)C, (int)M, (int)N, (int)nb, alpha,
                     (int)past_caches(C, M, N * sizeof(OutT), nb));
  return kamd_check(hipGetLastError(), "gemm_mxfp4_nt launch");
}

template <typename OutT, int NP, int NQ, int WAVES>
static int launch_rows_of(const void* P, const void* Ps, const void* Q, const void* Qs, void* C, int64_t np, int64_t nq,
                          int64_t nb, int64_t cp, int64_t cq, float alpha, Split split, hipStream_t stream) {
  constexpr int LDS = rows_lds(NP, NQ, WAVES);
  const int64_t tiles = ((np + NP * 16 - 1) / (NP * 16)) * ((nq + NQ * 16 - 1) / (NQ * 16));
  if (tiles * (WAVES * 64) >= (int64_t)1 << 32) return kamd_fail("gemm_mxfp4_nt: %lld x %lld is too large", (long long)np, (long long)nq);
  auto kernel = gemm_rows_kernel<OutT, NP, NQ, WAVES>;
  static std::atomic<uint64_t> asked{0};
  if (allow_lds(kernel, LDS, asked) != 0) return -1;
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, split.count), dim3(WAVES * 64), LDS, stream, (const uint8_t*)P,
                     (const uint8_t*)Ps, (const uint8_t*)Q, (const uint8_t*)Qs, (OutT*)C, (int)np, (int)nq, (int)nb, split.per,
                     cp, cq, alpha);
  return kamd_check(hipGetLastError(), "gemm_mxfp4_nt launch");
}

template <typename OutT>
static int launch_rows(const void* P, const void* Ps, const void* Q, const void* Qs, void* C, int64_t np, int64_t nq, int64_t nb,
                       int64_t cp, int64_t cq, float alpha, Split split, hipStream_t stream) {
  // Two tiles of P where one would make more than a workgroup for each CU: half the reads of Q, and one round
  // (16x5000x4096: 4.7 against 5.0 us, 32x5000x4096: 5.8 and 7.9). Eight waves where the workgroups are one for each
  // CU, whose LDS they fill; of more, with four, two lie on a CU (32x8192x8192: 8.9 against 10.0 us with four;
  // 32x10000x4096: 10.3 with eight and 8.8).
  const int64_t cus = 256, each = (nq + 15) / 16;
  const bool wide = np > 16 * cus;
  const bool many = (np + (wide ? 31 : 15)) / (wide ? 32 : 16) * (each <= 2 ? 1 : (each + 3) / 4) > cus;
#define KAMD_ROWS(NP, NQ, W) launch_rows_of<OutT, NP, NQ, W>(P, Ps, Q, Qs, C, np, nq, nb, cp, cq, alpha, split, stream)
  if (each == 1) {
    if (wide) return many ? KAMD_ROWS(2, 1, 4) : KAMD_ROWS(2, 1, 8);
    return KAMD_ROWS(1, 1, 8);
  }
  if (each == 2) {
    if (wide) return many ? KAMD_ROWS(2, 2, 4) : KAMD_ROWS(2, 2, 8);
    return KAMD_ROWS(1, 2, 8);
  }
  return wide ? KAMD_ROWS(2, 4, 4) : KAMD_ROWS(1, 4, 4);
#undef KAMD_ROWS
}

template <typename OutT>
static int launch_small(const void* A, const void* As, const void* B, const void* Bs, void* C, int64_t M, int64_t N, int64_t nb,
                        float alpha, bool tiles, Split split, hipStream_t stream) {
  if (tiles) return launch_tile<OutT, 1, 4>(A, As, B, Bs, C, M, N, nb, alpha, split, stream);
  // the operand with more rows is P; element (p, q) of the product at p * cp + q * cq
  return M <= N ? launch_rows<OutT>(B, Bs, A, As, C, N, M, nb, 1, N, alpha, split, stream)
                : launch_rows<OutT>(A, As, B, Bs, C, M, N, nb, N, 1, alpha, split, stream);
}

template <typename OutT>
static int launch_gemm(const void* A, const void* As, const void* B, const void* Bs, void* C, int64_t M, int64_t N, int64_t nb,
                       float alpha, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  const size_t n = (size_t)M * N;
  if (nb == 0) {
    return sliced(n, [&](size_t first, dim3 grid) {
      hipLaunchKernelGGL(zero_kernel<OutT>, grid, dim3(256), 0, stream, (OutT*)C, first, n);
    });
  }
  const int tile = tile_size(M, N, nb);
  if (tile == 256) return launch_large<OutT>(A, As, B, Bs, C, M, N, nb, alpha, workspace, workspace_bytes, stream);
  const Split split = split_k(M, N, nb);
  if (tile == 128)
    // one tile a CU: 4 stages; more: 2, and two tiles on a CU (2048x2048x8192: 25 and 30 us, 4096x2048x4096: 32 and 27)
    return ((M + 127) / 128) * ((N + 127) / 128) <= 256
               ? launch_tile<OutT, 2, 4>(A, As, B, Bs, C, M, N, nb, alpha, split, stream)
               : launch_tile<OutT, 2, 2>(A, As, B, Bs, C, M, N, nb, alpha, split, stream);
  if (split.count == 1) return launch_small<OutT>(A, As, B, Bs, C, M, N, nb, alpha, tile == 64, split, stream);
  const int64_t need = (int64_t)n * 4 * split.count;
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))
    return kamd_fail("gemm_mxfp4_nt: needs a workspace of %lld bytes, 16-byte aligned", (long long)need);
  if (launch_small<float>(A, As, B, Bs, workspace, M, N, nb, 1.f, tile == 64, split, stream) != 0) return -1;
  hipLaunchKernelGGL(join_kernel<OutT>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, (const float*)workspace, (OutT*)C, n,
                     split.count, alpha);
  return kamd_check(hipGetLastError(), "gemm_mxfp4_nt launch");
}
}  // namespace mxfp4

extern "C" {

// x: rows of K values (type 0 bf16, 1 fp16, 2 fp32), value k of row r at x + r * row_step + k * step elements, one of the
// two steps being 1; q: rows * 16 * nb bytes, 16-byte aligned; scale: rows * nb bytes
int kamd_mxfp4_quantize_launch(const void* x, void* q, void* scale, int64_t rows, int64_t K, int64_t row_step, int64_t step,
                               int type, hipStream_t stream) {
  using namespace mxfp4;
  if (rows < 0 || K < 0 || type < 0 || type > 2 || (step != 1 && row_step != 1 && K > 1))
    return kamd_fail("mxfp4_quantize: bad arguments");
  if (rows == 0 || K == 0) return 0;
  if (K >= LONGEST) return kamd_fail("mxfp4_quantize: K (%lld) is too large", (long long)K);
  const int64_t nb = (K + 31) / 32, row_items = nb * 4;
  if (!x || !q || !scale) return kamd_fail("mxfp4_quantize: a null pointer");
  if (((uintptr_t)q) & 15) return kamd_fail("mxfp4_quantize: codes must be 16-byte aligned");
  if (step != 1 && K > 1) {
    const int64_t tile = type == FP32 ? 64 : 128, tiles = (rows + tile - 1) / tile * ((nb + 7) / 8), most = SLICE / 512;
    auto k = type == BF16 ? quantize_cols_kernel<BF16> : type == FP16 ? quantize_cols_kernel<FP16> : quantize_cols_kernel<FP32>;
    for (int64_t first = 0; first < tiles; first += most) {
      hipLaunchKernelGGL(k, dim3((unsigned)(tiles - first < most ? tiles - first : most)), dim3(512), 0, stream, x, (uint8_t*)q,
                         (uint8_t*)scale, first, rows, K, step, nb);
      HC(hipGetLastError());
    }
    return 0;
  }
  if (row_items >= ROW_ITEMS)
    return pieces(rows, K, [&](int64_t r, int64_t k, int64_t n) {
      return kamd_mxfp4_quantize_launch((const char*)x + (r * row_step + k) * (type == FP32 ? 4 : 2), (char*)q + r * nb * 16 + k / 2,
                                        (char*)scale + r * nb + k / 32, 1, n, n, 1, type, stream);
    });
  const size_t items = (size_t)rows * row_items;
  return sliced(items, [&](size_t first, dim3 grid) {
    auto k = type == BF16 ? quantize_rows_kernel<BF16> : type == FP16 ? quantize_rows_kernel<FP16> : quantize_rows_kernel<FP32>;
    hipLaunchKernelGGL(k, grid, dim3(256), 0, stream, x, (uint32_t*)q, (uint8_t*)scale, first, items, (uint32_t)row_items, K,
                       row_step);
  });
}

// the inverse into contiguous rows of K values; q is 4-byte aligned
int kamd_mxfp4_dequantize_launch(const void* q, const void* scale, void* x, int64_t rows, int64_t K, int type,
                                 hipStream_t stream) {
  using namespace mxfp4;
  if (rows < 0 || K < 0 || type < 0 || type > 2) return kamd_fail("mxfp4_dequantize: bad arguments");
  if (rows == 0 || K == 0) return 0;
  if (K >= LONGEST) return kamd_fail("mxfp4_dequantize: K (%lld) is too large", (long long)K);
  const int64_t nb = (K + 31) / 32, row_items = nb * (type == FP32 ? 8 : 4);
  if (!q || !scale || !x) return kamd_fail("mxfp4_dequantize: a null pointer");
  if (((uintptr_t)q) & 3) return kamd_fail("mxfp4_dequantize: codes must be 4-byte aligned");
  if (row_items >= ROW_ITEMS)
    return pieces(rows, K, [&](int64_t r, int64_t k, int64_t n) {
      return kamd_mxfp4_dequantize_launch((const char*)q + r * nb * 16 + k / 2, (const char*)scale + r * nb + k / 32,
                                          (char*)x + (r * K + k) * (type == FP32 ? 4 : 2), 1, n, type, stream);
    });
  const size_t items = (size_t)rows * row_items;
  const bool stream_out = K * (type == FP32 ? 4 : 2) % 16 == 0 && ((uintptr_t)x & 15) == 0;
  return sliced(items, [&](size_t first, dim3 grid) {
    auto k = stream_out ? (type == BF16   ? dequantize_kernel<BF16, true>
                           : type == FP16 ? dequantize_kernel<FP16, true>
                                          : dequantize_kernel<FP32, true>)
                        : (type == BF16   ? dequantize_kernel<BF16, false>
                           : type == FP16 ? dequantize_kernel<FP16, false>
                                          : dequantize_kernel<FP32, false>);
    hipLaunchKernelGGL(k, grid, dim3(256), 0, stream, q, (const uint8_t*)scale, x, first, items, (uint32_t)row_items, K);
  });
}

// bytes of scratch memory that the product of these sizes needs, 0 for most
int64_t kamd_gemm_mxfp4_nt_workspace(int64_t M, int64_t N, int64_t nb) {
  if (M <= 0 || N <= 0 || nb <= 0) return 0;
  if (mxfp4::tile_size(M, N, nb) == 256) return mxfp4::arranged_bytes(M, N, nb);
  const int parts = mxfp4::split_k(M, N, nb).count;
  return parts > 1 ? (int64_t)parts * M * N * 4 : 0;
}

// C[M, N] = alpha * A B^T, A [M, 16 nb] / As [M, nb], B [N, 16 nb] / Bs [N, nb] contiguous, A and B 16-byte aligned;
// C fp32 or bf16, contiguous. nb = 0 gives zeros. The workspace is 16-byte aligned and used in stream order.
int kamd_gemm_mxfp4_nt_launch(const void* A, const void* As, const void* B, const void* Bs, void* C, int64_t M, int64_t N,
                              int64_t nb, float alpha, int out_fp32, void* workspace, int64_t workspace_bytes,
                              hipStream_t stream) {
  const int64_t most = (int64_t)1 << 27;
  if (M < 0 || N < 0 || nb < 0 || M > most || N > most || nb > most)
    return kamd_fail("gemm_mxfp4_nt: sizes out of range (%lld x %lld x %lld blocks)", (long long)M, (long long)N, (long long)nb);
  if (M == 0 || N == 0) return 0;
  if (!C || (nb != 0 && (!A || !As || !B || !Bs))) return kamd_fail("gemm_mxfp4_nt: a null pointer");
  if ((((uintptr_t)A) | ((uintptr_t)B)) & 15) return kamd_fail("gemm_mxfp4_nt: A/B must be 16-byte aligned");
  return out_fp32 ? mxfp4::launch_gemm<float>(A, As, B, Bs, C, M, N, nb, alpha, workspace, workspace_bytes, stream)
                  : mxfp4::launch_gemm<__bf16>(A, As, B, Bs, C, M, N, nb, alpha, workspace, workspace_bytes, stream);
}

// One sampled output of the fp4 burn-in, on the host: `got` = row A times row B, each row with its `size` bf16 values, codes
// and scales. Codes and scales have to be the definition's (else the error is 1), and `got` is held against the product of
// the codes in 64 bits, relative to the sum of magnitudes. *worst becomes the worse of itself and these.
int kamd_diag_mfma_fp4_sample(const uint16_t* xa, const uint8_t* qa, const uint8_t* sa, const uint16_t* xb, const uint8_t* qb,
                              const uint8_t* sb, int size, float got, double* worst) {
  if (size < 32 || size % 32 || !xa || !qa || !sa || !xb || !qb || !sb || !worst) return kamd_fail("diag_mfma_fp4_sample: bad arguments");
  static const double grid[8] = {0, 0.5, 1, 1.5, 2, 3, 4, 6};
  bool exact = true;
  auto block = [&](const uint16_t* x, const uint8_t* q, int scale, double* v) {   // the values of 32 codes
    double in[32], top = 0;
    bool finite = true;
    for (int k = 0; k < 32; ++k) {
      const uint32_t u = (uint32_t)x[k] << 16;
      float f;
      memcpy(&f, &u, 4);
      in[k] = f;
      finite &= std::isfinite(f);
      if (fabs(in[k]) > top) top = fabs(in[k]);
    }
    const int s = !finite ? 255 : top == 0 || ilogb(top) < 2 - 127 ? 0 : ilogb(top) - 2 + 127;
    exact &= s == scale;
    for (int k = 0; k < 32; ++k) {
      const int code = (q[k / 2] >> (k % 2 * 4)) & 15;
      const double w = fabs(ldexp(in[k], 127 - s));
      const int want = (w > 0.25) + (w >= 0.75) + (w > 1.25) + (w >= 1.75) + (w > 2.5) + (w >= 3.5) + (w > 5) + (std::signbit(in[k]) ? 8 : 0);
      exact &= code == (finite ? want : 0);
      v[k] = scale == 255 ? NAN : ldexp(code & 8 ? -grid[code & 7] : grid[code & 7], scale - 127);
    }
  };
  double ref = 0, mag = 0;
  for (int b = 0; b < size / 32; ++b) {
    double va[32], vb[32];
    block(xa + b * 32, qa + b * 16, sa[b], va);
    block(xb + b * 32, qb + b * 16, sb[b], vb);
    for (int k = 0; k < 32; ++k) {
      ref += va[k] * vb[k];
      mag += fabs(va[k] * vb[k]);
    }
  }
  *worst = kamd_worse(kamd_worse(*worst, exact ? 0 : 1), fabs(got - ref) / (mag > 1e-30 ? mag : 1.0));
  return 0;
}

// fp4 burn-in, the protocol of kamd_diag_mfma: random bf16 operands of size x size are quantised on the device, then
// `iters` products timed, and 256 outputs checked with their rows. size is a multiple of 32.
int kamd_diag_mfma_fp4(int dev, int size, int iters, double* tflops, double* max_rel_err) {
  using namespace mxfp4;
  if (size < 32 || size % 32 || iters < 1)
    return kamd_fail("diag_mfma_fp4: size (%d) must be a multiple of 32, iterations (%d) at least 1", size, iters);
  HC(hipSetDevice(dev));
  const size_t n = size, nb = n / 32;
  uint8_t* mem = nullptr;   // x | codes of A, B | C | scales of A, B | workspace
  const size_t at_q = n * n * 2 * 2, at_c = at_q + n * n, at_s = at_c + n * n * 4, at_w = (at_s + 2 * n * nb + 255) & ~(size_t)255;
  const int64_t ws = kamd_gemm_mxfp4_nt_workspace(size, size, (int64_t)nb);
  HC(hipMalloc(&mem, at_w + ws));
  uint8_t *qa = mem + at_q, *qb = qa + n * n / 2, *sa = mem + at_s, *sb = sa + n * nb;
  float* c = (float*)(mem + at_c);
  uint16_t* x = (uint16_t*)mem;
  hipEvent_t e0 = nullptr, e1 = nullptr;
  int rc = -1;
  try {
    do {
      hipLaunchKernelGGL(fill_kernel, dim3(1024), dim3(256), 0, 0, x, 2 * n * n);
      if (kamd_check(hipGetLastError(), "diag_mfma_fp4 fill") != 0) break;
      if (kamd_mxfp4_quantize_launch(x, qa, sa, size, size, size, 1, BF16, 0) != 0) break;
      if (kamd_mxfp4_quantize_launch(x + n * n, qb, sb, size, size, size, 1, BF16, 0) != 0) break;
      auto product = [&] {
        return kamd_gemm_mxfp4_nt_launch(qa, sa, qb, sb, c, size, size, (int64_t)nb, 1.f, 1, ws ? mem + at_w : nullptr, ws, 0);
      };
      if (product() != 0) break;   // warm-up
      if (kamd_check(hipEventCreate(&e0), "diag_mfma_fp4 event") != 0 || kamd_check(hipEventCreate(&e1), "diag_mfma_fp4 event") != 0) break;
      if (kamd_check(hipEventRecord(e0, 0), "diag_mfma_fp4 event") != 0) break;
      bool ok = true;
      for (int i = 0; i < iters && ok; ++i) ok = product() == 0;
      if (!ok) break;
      if (kamd_check(hipEventRecord(e1, 0), "diag_mfma_fp4 event") != 0) break;
      if (kamd_check(hipEventSynchronize(e1), "diag_mfma_fp4 sync") != 0) break;
      float ms = 0.f;
      if (kamd_check(hipEventElapsedTime(&ms, e0, e1), "diag_mfma_fp4 time") != 0) break;
      *tflops = 2.0 * size * size * (double)size * iters / (ms * 1e-3) / 1e12;

      double worst = 0;
      struct Row {
        std::vector<uint16_t> x;
        std::vector<uint8_t> q, s;
      } a, b;
      auto fetch = [&](Row& to, const uint16_t* x, const uint8_t* q, const uint8_t* s) {
        to.x.resize(n);
        to.q.resize(n / 2);
        to.s.resize(nb);
        return kamd_check(hipMemcpy(to.x.data(), x, n * 2, hipMemcpyDeviceToHost), "diag_mfma_fp4 copy") == 0 &&
               kamd_check(hipMemcpy(to.q.data(), q, n / 2, hipMemcpyDeviceToHost), "diag_mfma_fp4 copy") == 0 &&
               kamd_check(hipMemcpy(to.s.data(), s, nb, hipMemcpyDeviceToHost), "diag_mfma_fp4 copy") == 0;
      };
      for (int t = 0; t < 256 && ok; ++t) {
        const size_t i = (size_t)t * 7919u % n, j = ((size_t)t * 104729u + 13u) % n;
        float got = 0;
        ok = fetch(a, x + i * n, qa + i * n / 2, sa + i * nb) && fetch(b, x + (n + j) * n, qb + j * n / 2, sb + j * nb) &&
             kamd_check(hipMemcpy(&got, c + i * n + j, 4, hipMemcpyDeviceToHost), "diag_mfma_fp4 copy") == 0 &&
             kamd_diag_mfma_fp4_sample(a.x.data(), a.q.data(), a.s.data(), b.x.data(), b.q.data(), b.s.data(), size, got, &worst) == 0;
      }
      if (!ok) break;
      *max_rel_err = worst;
      rc = 0;
    } while (0);
  } catch (const std::exception& e) {   // no memory on the host
    kamd_fail("diag_mfma_fp4: %s", e.what());
    rc = -1;
  }
  if (e0) (void)hipEventDestroy(e0);
  if (e1) (void)hipEventDestroy(e1);
  (void)hipFree(mem);
  return rc;
}

}  // extern "C"
