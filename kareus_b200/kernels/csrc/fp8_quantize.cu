// bf16 → 8-bit floating point with power-of-two scales, along the rows, along the columns, or both in one pass.
//
// A piece of 128 elements along the contraction (of 128 x 128 for a weight, so that the same values serve as the weight and as its
// transpose) is held as q * 2^E: E is the smallest integer with |x| <= max * 2^E over the piece (max: 448 for e4m3, 57344 for
// e5m2), q the nearest value of the format, ties to even.  A scale is one byte, E + 127; it is read off the bits of the largest
// |x|, so nothing here is rounded but q itself: x * 2^-E is exact in fp32.  A piece of zeros has the byte 0.  A piece with an
// infinity or a NaN has the byte 255 (NaN) and stands for NaN as a whole: an overflow stays visible and does not become a large
// number.
//
// Scales are laid out as the product's tensor memory takes them (gemm_fp8_sm100.cu): 128 rows x 4 pieces are 512 bytes, row r of
// them at (r % 32) * 16 + (r / 32) * 4; [ceil(rows / 128)][ceil(pieces / 4)] such blocks.  Bytes past the edge are 0.
//
// What bounds it: memory.  A block of 256 threads takes a 128 x 128 tile, reads it once (16 lanes a row, 16 bytes each), writes the
// rows' bytes from registers and the columns' by way of shared memory, in whole lines of 128 tokens (as 32-byte pieces of a thread
// each they took a third longer).  One B200: 8192 x 14336 along both 82 us, 5.7 TB/s; 6144 x 4096 with 128 x 128 scales, rows only, 15.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "launch.h"
#include "native_ops.h"
#include "pdl.cuh"

namespace kb {

struct Fp8Quantize {
  const __nv_bfloat16* x;
  long ld;                      // elements from row to row
  int rows, cols;
  uint8_t *q, *s;               // [rows, ldq] and its scales; null: not wanted
  uint8_t *qt, *st;             // [cols, ldqt] (the transpose) and its scales; null: not wanted
  long ldq, ldqt;
  int tiles_c;                  // 128-column tiles
  bool vec;                     // rows start on 16 bytes and hold whole 16-byte units
};

constexpr int FQ_THREADS = 256;
constexpr int FQ_PITCH = 68;    // words from row to row of the staged tile: rows start on 16 bytes, units of a row on other banks

// Scale byte of a piece whose largest |x| has these bf16 bits; TOP: the format's largest value is 0.875 * 2^TOP.
template <int TOP>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  const int e = static_cast<int>(amax >> 7);
  if (e == 255) return 255u;
  const int b = e + 1 - TOP + ((amax & 127u) > 96u ? 1 : 0);    // 1.mmmmmmm > 1.75 does not fit any more
  return b > 0 ? static_cast<uint32_t>(b) : 0u;
}
// 2^-E
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : (254u - byte) << 23);
}
// Four values as four bytes, the first in the lowest.
template <bool E5M2>
__device__ __forceinline__ uint32_t quantize4(float a, float b, float c, float d) {
  uint32_t r;
  if constexpr (E5M2)
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e5m2x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e5m2x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
        : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  else
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
        : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// The two bf16 of a word, each times its factor.
__device__ __forceinline__ float2 scaled(uint32_t v, float2 inv) {
  return __fmul2_rn(make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)), inv);
}
// Larger |x| of two pairs of bf16, element by element; a NaN stays one.  The signs of the result mean nothing.
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}

// Where the scale of (row, piece) lies.
__device__ __forceinline__ size_t scale_at(int row, int piece, int groups) {
  return (static_cast<size_t>(row >> 7) * groups + (piece >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (piece & 3);
}
// Writes it; the last piece also clears what is left of its group of four.
__device__ __forceinline__ void put_scale(uint8_t* s, int row, int piece, int pieces, uint32_t byte) {
  const int groups = (pieces + 3) >> 2;
  s[scale_at(row, piece, groups)] = static_cast<uint8_t>(byte);
  if (piece == pieces - 1)
    for (int p = pieces; p & 3; ++p) s[scale_at(row, p, groups)] = 0;
}

template <bool E5M2, bool SQUARE>
__global__ void __launch_bounds__(FQ_THREADS, 4) fp8_quantize_kernel(const Fp8Quantize p) {
  __shared__ __align__(16) uint32_t tile[128 * FQ_PITCH];
  __shared__ uint32_t part[4][64];
  __shared__ uint32_t whole[FQ_THREADS / 32];
  __shared__ uint8_t row_byte[128], col_byte[128];
  constexpr int TOP = E5M2 ? 16 : 9;
  pdl_begin();
  const int tr = blockIdx.x / p.tiles_c, tc = blockIdx.x - tr * p.tiles_c;
  const int r0 = tr * 128, c0 = tc * 128;
  const int tid = threadIdx.x, unit = tid & 15, rsub = tid >> 4;
  const int col = c0 + unit * 8;
  uint4 v[8];                                   // rows r0 + rsub + 16 i, columns col .. col + 7
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = r0 + i * 16 + rsub;
    v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (row < p.rows && col < p.cols) {
      const __nv_bfloat16* src = p.x + row * p.ld + col;
      if (p.vec) {
        v[i] = __ldcs(reinterpret_cast<const uint4*>(src));
      } else {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j < p.cols) w[j >> 1] |= static_cast<uint32_t>(__bfloat16_as_ushort(src[j])) << (j & 1 ? 16 : 0);
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  uint32_t block_byte = 0;
  if constexpr (SQUARE) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_abs2(m, max_abs2(max_abs2(v[i].x, v[i].y), max_abs2(v[i].z, v[i].w)));
    m = max(m & 0x7fffu, m >> 16 & 0x7fffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if ((tid & 31) == 0) whole[tid >> 5] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int i = 0; i < FQ_THREADS / 32; ++i) m = max(m, whole[i]);
    block_byte = scale_byte<TOP>(m);
  }
  if (p.q) {
    uint32_t byte[8];
    if constexpr (!SQUARE) {
      // two rows' maxima in a word, over the 16 lanes that hold the rows
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const uint32_t a = max_abs2(max_abs2(v[i].x, v[i].y), max_abs2(v[i].z, v[i].w));
        const uint32_t b = max_abs2(max_abs2(v[i + 1].x, v[i + 1].y), max_abs2(v[i + 1].z, v[i + 1].w));
        uint32_t m = max_abs2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
        for (int s = 8; s > 0; s >>= 1) m = max_abs2(m, __shfl_xor_sync(0xffffffffu, m, s));
        byte[i] = scale_byte<TOP>(m & 0x7fffu);
        byte[i + 1] = scale_byte<TOP>(m >> 16 & 0x7fffu);
      }
    }
    uint8_t* dst = p.q + (r0 + rsub) * p.ldq + col;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (SQUARE) byte[i] = block_byte;
      const float f = inverse_scale(byte[i]);
      const float2 inv = make_float2(f, f);
      const float2 a = scaled(v[i].x, inv), b = scaled(v[i].y, inv), c = scaled(v[i].z, inv), d = scaled(v[i].w, inv);
      const uint2 o = make_uint2(quantize4<E5M2>(a.x, a.y, b.x, b.y), quantize4<E5M2>(c.x, c.y, d.x, d.y));
      if (r0 + i * 16 + rsub < p.rows && col < p.ldq) *reinterpret_cast<uint2*>(dst) = o;
      dst += 16 * p.ldq;
      if (unit == 0) row_byte[i * 16 + rsub] = static_cast<uint8_t>(byte[i]);
    }
  }
  if (p.qt) {
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(tile + (i * 16 + rsub) * FQ_PITCH + unit * 4) = v[i];
    __syncthreads();
    const int pair = tid & 63, rg = tid >> 6;             // two columns, 32 rows
    uint32_t w[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) w[j] = tile[(rg * 32 + j) * FQ_PITCH + pair];
    uint32_t b0 = block_byte, b1 = block_byte;
    if constexpr (!SQUARE) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 32; ++j) m = max_abs2(m, w[j]);
      part[rg][pair] = m;
      __syncthreads();
      m = max_abs2(max_abs2(part[0][pair], part[1][pair]), max_abs2(part[2][pair], part[3][pair]));
      b0 = scale_byte<TOP>(m & 0x7fffu);
      b1 = scale_byte<TOP>(m >> 16 & 0x7fffu);
    }
    if (rg == 0) {
      col_byte[2 * pair] = static_cast<uint8_t>(b0);
      col_byte[2 * pair + 1] = static_cast<uint8_t>(b1);
    }
    if constexpr (SQUARE) __syncthreads();                // (else the one above) everybody has read the tile
    // The columns' bytes go through its place, so that a column's 128 leave as whole lines: 16-byte units, swizzled by column pair.
    const float2 inv = make_float2(inverse_scale(b0), inverse_scale(b1));
    uint4* const bytes = reinterpret_cast<uint4*>(tile);  // [128 columns][8 units]
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t lo[4], hi[4];                              // 16 rows of either column
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t* x = w + half * 16 + 4 * j;
        const float2 e = scaled(x[0], inv), f = scaled(x[1], inv), g = scaled(x[2], inv), h = scaled(x[3], inv);
        lo[j] = quantize4<E5M2>(e.x, f.x, g.x, h.x);
        hi[j] = quantize4<E5M2>(e.y, f.y, g.y, h.y);
      }
      const int at = (rg * 2 + half) ^ (pair & 7);
      bytes[2 * pair * 8 + at] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      bytes[(2 * pair + 1) * 8 + at] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    }
    __syncthreads();
    const int cu = tid & 7;                               // ldqt is a multiple of 16: 16-byte units are whole or outside
    if (r0 + cu * 16 < p.ldqt) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = k * 32 + (tid >> 3);
        if (c0 + c < p.cols) *reinterpret_cast<uint4*>(p.qt + (c0 + c) * p.ldqt + r0 + cu * 16) = bytes[c * 8 + (cu ^ ((c >> 1) & 7))];
      }
    }
  }
  __syncthreads();
  const int i = tid & 127;
  if (tid < 128) {
    if (p.q) put_scale(p.s, r0 + i, tc, p.tiles_c, r0 + i < p.rows ? row_byte[i] : 0u);
  } else if (p.qt) {
    put_scale(p.st, c0 + i, tr, (p.rows + 127) >> 7, c0 + i < p.cols ? col_byte[i] : 0u);
  }
}

}  // namespace kb

// x: [rows, cols] bf16, `ld` elements from row to row.  q [rows, ldq] / s and qt [cols, ldqt] / st: see above, either pair null.
// ldq and ldqt are multiples of 16, at least cols / rows; what lies between the two is nobody's.  fmt: 0 e4m3, 1 e5m2.
extern "C" int kb_fp8_quantize(const void* x, long rows, long cols, long ld, void* q, long ldq, void* s, void* qt, long ldqt,
                               void* st, int square, int fmt, cudaStream_t stream) {
  constexpr long MOST = (1L << 31) - 512;       // row and column numbers are ints, those of tiles across the edge too
  if (rows <= 0 || cols <= 0 || rows > MOST || cols > MOST || ld < cols || (!q && !qt) || (fmt & ~1)) return 7;
  if (q && (!s || ldq < cols || ldq % 16 || reinterpret_cast<uintptr_t>(q) % 16)) return 7;
  if (qt && (!st || ldqt < rows || ldqt % 16 || reinterpret_cast<uintptr_t>(qt) % 16)) return 7;
  kb::Fp8Quantize p;
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.ld = ld;
  p.rows = static_cast<int>(rows);
  p.cols = static_cast<int>(cols);
  p.q = static_cast<uint8_t*>(q);
  p.s = static_cast<uint8_t*>(s);
  p.qt = static_cast<uint8_t*>(qt);
  p.st = static_cast<uint8_t*>(st);
  p.ldq = ldq;
  p.ldqt = ldqt;
  p.tiles_c = static_cast<int>((cols + 127) / 128);
  p.vec = cols % 8 == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  const long blocks = (rows + 127) / 128 * p.tiles_c;
  if (blocks >= 1L << 31) return 7;
  auto kern = fmt ? (square ? kb::fp8_quantize_kernel<true, true> : kb::fp8_quantize_kernel<true, false>)
                  : (square ? kb::fp8_quantize_kernel<false, true> : kb::fp8_quantize_kernel<false, false>);
  KB_LAUNCH_PDL(kern, static_cast<unsigned>(blocks), kb::FQ_THREADS, 0, stream, p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 2000 + static_cast<int>(e);
}
