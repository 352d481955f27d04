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
#include <type_traits>
#include <utility>
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
typedef float f32x16 __attribute__((ext_vector_type(16)));
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

// Tile of workgroup w. Workgroups go to the 8 XCDs in turn; each XCD gets a run of consecutive tiles, and a run
// walks groups of GROUP tile rows down and then right, so that what is in an XCD's L2 is used by its neighbours.
__device__ __forceinline__ void tile_of(uint32_t w, int tiles_m, int tiles_n, int& tm, int& tn) {
  constexpr uint32_t GROUP = 4;
  const uint32_t n = (uint32_t)tiles_m * tiles_n, x = w & 7, q = n >> 3, rest = n & 7;
  const uint32_t t = x * q + min(x, rest) + (w >> 3);
  const uint32_t in_group = GROUP * tiles_n, first = t / in_group * GROUP, rows = min((uint32_t)tiles_m - first, GROUP);
  tm = (int)(first + t % in_group % rows);
  tn = (int)(t % in_group / rows);
}

// ---------------------------------------------------------------------------
// Large products. A workgroup of 4 waves makes a BM x BN tile of C, each wave a quarter of TM x TN tiles of
// 32x32 (v_mfma_scale_f32_32x32x64_f8f6f4: lane l holds chunk l / 32 of row l % 32 and that block's scale).
// K goes by in tiles of 8 blocks (256 values, 128 B a row), two of them in LDS:
//   * codes HBM -> LDS without registers (global_load_lds, 16 B a lane), 16-byte slot s of row r holding chunk
//     s ^ (r / 2 % 8), so that 16 rows' reads of one chunk meet all 64 banks once;
//   * step s = 0 .. 3 of a tile gives lane l the chunk 4 (l / 32) + s: its four scales are neighbours, one
//     32-bit word, which the instruction's byte select takes apart;
//   * scales HBM -> registers -> LDS as [row % 32][half][row / 32], so that a lane has those of all its rows of
//     a tile in one read. Rows of scales are read at any byte alignment.
// While a step's products run, the next step's fragments are read into the other register set; the one barrier
// of a tile stands before its last step, where its last read has returned and the next tile has arrived.
// B's rows are the instruction's rows, A's its columns: a lane ends with 4 neighbours of a row of C.
// Tiles at the lower and right edge are moved up and left into C; what two tiles cover both write alike.
template <int N, typename F, int... I>
__device__ __forceinline__ void unroll_(F f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, typename F>
__device__ __forceinline__ void unroll(F f) { unroll_<N>(f, std::make_integer_sequence<int, N>{}); }

typedef __attribute__((address_space(3))) void lds_void;

template <int T> struct Scales { uint32_t v[T]; };   // of T row groups, 4 blocks each

constexpr int tile_lds(int BM, int BN) { return 2 * (BM + BN) * (128 + 8); }

// acc += a b^T with byte S of the scales. ACC: in place in the accumulation registers. The compiler's own form
// gives the sum another place and moves it back, which with 256 of them costs more than the products. What
// inline assembly has to see to: 2 wait states after an ordinary instruction's write of an operand (the s_nop),
// and the wait before a sum is read (settle). Sums are used again 16 instructions later, after any wait there is.
template <bool ACC, int S>
__device__ __forceinline__ void mfma32(f32x16& acc, i32x4 a, i32x4 b, uint32_t sa, uint32_t sb) {
  if constexpr (ACC) {
    asm volatile(
        "s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%5,0] op_sel_hi:[%6,%6,0] cbsz:4 blgp:4"
        : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb), "i"(S & 1), "i"(S >> 1));
  } else {
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(frag(a), frag(b), acc, 4, 4, S, (int)sa, S, (int)sb);
  }
}
template <bool ACC>
__device__ __forceinline__ void settle(f32x16& acc) {
  if constexpr (ACC) asm volatile("s_nop 15\n\ts_nop 15" : "+a"(acc));
}

template <typename OutT, int TM, int TN>
__global__ void __launch_bounds__(256, TM == 4 ? 1 : 2)
gemm_tile_kernel(const uint8_t* __restrict__ A, const uint8_t* __restrict__ As, const uint8_t* __restrict__ B,
                 const uint8_t* __restrict__ Bs, OutT* __restrict__ C, int M, int N, int nb, float alpha) {
  constexpr int BM = 64 * TM, BN = 64 * TN;
  constexpr int DATA = (BM + BN) * 128, SCALE = (BM + BN) * 8;
  constexpr bool ACC = TM * TN == 16;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // 2 x codes of A, B; 2 x scales of A, B
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int wm = wave >> 1, wn = wave & 1;
  int tm, tn;
  tile_of(blockIdx.x, (M + BM - 1) / BM, (N + BN - 1) / BN, tm, tn);
  const int m0 = min(tm * BM, M - BM), n0 = min(tn * BN, N - BN);
  const int nt = (nb + 7) / 8, rem = nb - (nt - 1) * 8;   // tiles of K, blocks of the last

  // staging: a wave's load takes 8 rows of 128 B, and 32 rows on with the next
  const size_t row_bytes = (size_t)nb * 16;
  const int srow = wave * 8 + (lane >> 3), chunk = (lane & 7) ^ ((srow >> 1) & 7);
  const uint32_t off = (uint32_t)srow * (uint32_t)row_bytes + chunk * 16;
  const uint8_t* const tA = A + (size_t)m0 * row_bytes;
  const uint8_t* const tB = B + (size_t)n0 * row_bytes;
  constexpr int LOADS = (BM + BN) / 32;
  auto stage = [&](int t, int j, auto last) {
    uint32_t o = off;
    if (last && chunk >= rem) o -= (uint32_t)(chunk - rem + 1) * 16;   // behind the last block: that one again
    const uint8_t* p = (j < BM / 32 ? tA + j * 32 * row_bytes : tB + (j - BM / 32) * 32 * row_bytes) + (size_t)t * 128;
    __builtin_amdgcn_global_load_lds((const void*)(p + o), (lds_void*)(lds + (t & 1) * DATA + wave * 1024 + j * 4096), 16, 0, 0);
  };

  // scales: a thread takes 8 bytes of a row. Of a short last tile those that end with the row, moved down.
  constexpr int NS = (BM + BN + 255) / 256;
  uint64_t sreg[NS];
  const uint8_t* sp[NS];
  uint32_t sw[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const int q = min(wave * 64 + n * 256, BM + BN - 64) + lane;   // a wave without rows repeats the last ones
    const bool isA = q < BM;
    const int row = isA ? q : q - BM, T = isA ? TM : TN;
    sp[n] = (isA ? As + (size_t)(m0 + row) * nb : Bs + (size_t)(n0 + row) * nb);
    sw[n] = 2 * DATA + (isA ? 0 : BM * 8) + row / (32 * T) * (256 * T) + (row & 31) * (8 * T) + row / 32 % T * 4;
  }
  auto sload = [&](int t, auto last) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      __builtin_memcpy(&sreg[n], sp[n] + (size_t)t * 8 - (last ? 8 - rem : 0), 8);
      if (last) sreg[n] >>= 8 * (8 - rem);
    }
  };
  auto swrite = [&](int t) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int T = min(wave * 64 + n * 256, BM + BN - 64) < BM ? TM : TN;
      *(uint32_t*)(lds + sw[n] + (t & 1) * SCALE) = (uint32_t)sreg[n];
      *(uint32_t*)(lds + sw[n] + (t & 1) * SCALE + 4 * T) = (uint32_t)(sreg[n] >> 32);
    }
  };

  // fragments
  const int baseA = (wm * 32 * TM + r) * 128, baseB = BM * 128 + (wn * 32 * TN + r) * 128;
  struct Frags { i32x4 a[TM], b[TN]; } f[2];
  static_assert(TM == TN, "fragments of A and B are read in pairs");
  // Fragments of step s, two at a time, asked for in the first groups of the step before: the last of them is on its
  // way while the other groups' products run.
  auto read = [&](int t, auto s, int pair) {
    if (2 * pair >= TM + TN) return;
#pragma unroll
    for (int k = 2 * pair; k < 2 * pair + 2; ++k) {
      const uint8_t* p = lds + (t & 1) * DATA + (((4 * h + s) ^ ((r >> 1) & 7)) << 4);
      if (k % 2 == 0) f[s % 2].b[k / 2] = *(const i32x4*)(p + baseB + k / 2 * 4096);
      else f[s % 2].a[k / 2] = *(const i32x4*)(p + baseA + k / 2 * 4096);
    }
  };
  Scales<TM> sa;
  Scales<TN> sb;
  auto sread = [&](int t) {
    const uint8_t* p = lds + 2 * DATA + (t & 1) * SCALE + wm * (256 * TM) + (r * 2 + h) * 4 * TM;
    __builtin_memcpy(&sa, __builtin_assume_aligned(p, 4 * TM), sizeof sa);
    p = lds + 2 * DATA + (t & 1) * SCALE + BM * 8 + wn * (256 * TN) + (r * 2 + h) * 4 * TN;
    __builtin_memcpy(&sb, __builtin_assume_aligned(p, 4 * TN), sizeof sb);
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  // Step s on one register set, in TM + TN groups: some of the products, then ask(k) asks for something. Asked
  // for before the first product, it would be in what that product waits for.
  auto step = [&](auto s, const Scales<TM>& ua, const Scales<TN>& ub, auto ask) {
    constexpr int GROUPS = TM + TN;
    unroll<GROUPS>([&](auto k) {
      unroll<TM * TN>([&](auto p) {
        if constexpr (p * GROUPS / (TM * TN) == k)
          mfma32<ACC, s>(acc[p / TN][p % TN], f[s % 2].b[p % TN], f[s % 2].a[p / TN], ub.v[p % TN], ua.v[p / TN]);
      });
      __builtin_amdgcn_sched_barrier(0);
      ask(k);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto landed = [] {   // what this wave asked for is in LDS, what it read is in registers; then everyone's
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
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

  // a tile with another behind it; the tile after that is asked for in the last step
  auto tile = [&](int t, auto fetch, auto last) {
    step(s0, sa, sb, [&](auto k) { read(t, s1, k); });
    step(s1, sa, sb, [&](auto k) { read(t, s2, k); });
    step(s2, sa, sb, [&](auto k) { read(t, s3, k); });
    swrite(t + 1);
    landed();
    const Scales<TM> ua = sa;
    const Scales<TN> ub = sb;
    step(s3, ua, ub, [&](auto k) {
      if constexpr (k == 0) sread(t + 1);
      read(t + 1, s0, k);
      if constexpr (fetch) {
        stage(t + 2, 2 * k, last);
        stage(t + 2, 2 * k + 1, last);
        if constexpr (k == TM + TN - 1) sload(t + 2, last);
      }
    });
  };
  auto fetch = [&](int t, auto last) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) stage(t, j, last);
    sload(t, last);
  };

  fetch(0, no);
  swrite(0);
  landed();
  if (nt > 2) fetch(1, no);
  else if (nt == 2) fetch(1, yes);
  unroll<TM + TN>([&](auto k) { read(0, s0, k); });
  sread(0);
  int t = 0;
  for (; t < nt - 3; ++t) tile(t, yes, no);
  if (t < nt - 2) tile(t++, yes, yes);
  if (t < nt - 1) tile(t++, no, no);
  // the last tile: what is behind the last block is multiplied by zeros
  auto clear = [&](auto s) {
    if (4 * h + s >= rem) {
#pragma unroll
      for (int i = 0; i < TM; ++i) f[s % 2].a[i] = i32x4{0, 0, 0, 0};
    }
  };
  clear(s0);
  step(s0, sa, sb, [&](auto k) { read(t, s1, k); });
  clear(s1);
  step(s1, sa, sb, [&](auto k) { read(t, s2, k); });
  clear(s2);
  step(s2, sa, sb, [&](auto k) { read(t, s3, k); });
  clear(s3);
  step(s3, sa, sb, [&](auto) {});

  // element e of lane (r, h): column r, row 8 (e / 4) + 4 h + e % 4
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    OutT* p = C + (size_t)(m0 + wm * 32 * TM + i * 32 + r) * N + n0 + wn * 32 * TN + h * 4;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      settle<ACC>(acc[i][j]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        OutT v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (OutT)(alpha * acc[i][j][q * 4 + e]);
        __builtin_memcpy(p + j * 32 + q * 8, v, sizeof v);
      }
    }
  }
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

template <typename OutT, int T>
static int launch_tile_of(const void* A, const void* As, const void* B, const void* Bs, void* C, int64_t M, int64_t N,
                          int64_t nb, float alpha, hipStream_t stream) {
  constexpr int BM = 64 * T, LDS = tile_lds(BM, BM);
  // what the kernel's addresses assume: whole tiles inside C, 8 blocks to read, 32-bit offsets in a tile
  if (M < BM || N < BM || nb < 8 || nb > 1 << 20) return kamd_fail("gemm_mxfp4_nt: no tile of %d in %lld x %lld x %lld blocks", BM, (long long)M, (long long)N, (long long)nb);
  // more than 64 KiB of LDS has to be asked for, on every device that the kernel runs on
  if (LDS > 64 * 1024)
    HC(hipFuncSetAttribute((const void*)gemm_tile_kernel<OutT, T, T>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
  const int64_t tiles = ((M + BM - 1) / BM) * ((N + BM - 1) / BM);
  if (tiles >= (int64_t)1 << 24) return kamd_fail("gemm_mxfp4_nt: %lld x %lld is too large", (long long)M, (long long)N);
  hipLaunchKernelGGL((gemm_tile_kernel<OutT, T, T>), dim3((unsigned)tiles), dim3(256), LDS, stream, (const uint8_t*)A,
                     (const uint8_t*)As, (const uint8_t*)B, (const uint8_t*)Bs, (OutT*)C, (int)M, (int)N, (int)nb, alpha);
  return kamd_check(hipGetLastError(), "gemm_mxfp4_nt launch");
}

template <typename OutT>
static int launch_tile(int T, const void* A, const void* As, const void* B, const void* Bs, void* C, int64_t M, int64_t N,
                       int64_t nb, float alpha, hipStream_t stream) {
  switch (T) {
    case 1: return launch_tile_of<OutT, 1>(A, As, B, Bs, C, M, N, nb, alpha, stream);
    case 2: return launch_tile_of<OutT, 2>(A, As, B, Bs, C, M, N, nb, alpha, stream);
    default: return launch_tile_of<OutT, 4>(A, As, B, Bs, C, M, N, nb, alpha, stream);
  }
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
  if (nb >= 8 && nb <= 1 << 20 && M >= 64 && N >= 64) {
    // ROUTE
    const int cus = 256;
    int T = 1;
    if (M >= 128 && N >= 128 && ((M + 127) / 128) * ((N + 127) / 128) >= cus) T = 2;
    if (M >= 256 && N >= 256 && ((M + 255) / 256) * ((N + 255) / 256) >= cus) T = 4;
    return out_fp32 ? launch_tile<float>(T, A, As, B, Bs, C, M, N, nb, alpha, stream)
                    : launch_tile<__bf16>(T, A, As, B, Bs, C, M, N, nb, alpha, stream);
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
