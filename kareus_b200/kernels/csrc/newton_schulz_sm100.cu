// Orthogonalising matrices by Newton-Schulz products, and the optimizer step built on it (Muon).
//
// X_0 = U / (|U|_F + eps), then a number of times
//     G = X Xt,   P = b G + c G G,   X <- a X + P X          (matrices with more rows than columns: G = Xt X, X <- a X + X P)
// which takes the singular values s of X to a s + b s^3 + c s^5 and leaves the singular vectors.
//
// Types.  The products run on the tensor cores in fp16 with fp32 sums: their operands are bounded by the singular values, so fp16
// with a common power of two (`scale`, chosen by the host so that the largest possible entry fits) has 11 bits for everything that
// counts where bf16 has 8.  Five steps, relative 2-norm against 64 bits, the result's rounding to bf16 (1.7e-3) included: 1.7e-3 to
// 2.1e-3 for matrices of one size of singular values (products in bf16: 2e-2 to 5e-2), 4e-3 to 6e-3 for singular values over three
// decades (7e-2), 6e-3 to 1e-2 over six (0.1): rounding X_0 puts 1.4e-4 of its norm in all directions, and the steps make what is small
// up to 3.4445^5 = 485 times as large.  Matrices of a few rows and columns whose smallest singular value is by chance below 1e-3 of
// the largest are up to 9e-2 off (2 x 2), 9e-3 (16 x 16).  The largest rounding errors would be those of
// the square matrices' diagonals (about 1 and -2.6 beside entries near 0, and much the same in every row), so diagonals are also kept
// in fp32: P's apart from P (X <- (a + diag P) X + (P - diag P) X), the others beside the matrix, where they put right what its
// rounded diagonal does to the result's.  Norms are summed in fp32 per thread and fp64 beyond, in a fixed order.
//
// Long matrices.  X_{k+1} = Q_k X_k with Q_k = a I + P_k, and G_{k+1} = Q_k G_k Q_k, where everything but X is as small as the shorter
// side.  Where the longer side is at least 1.5 times the shorter one and it saves time (ns_carries), G is carried from step to step
// so (T = Q G, G' = Q T), the Q are multiplied up, and X is read twice per segment of two or three steps instead of twice per step:
// five steps of a matrix with sides m and r m take 6 r + 14 units of m^3 multiplications instead of 15 r + 5.  G of a carried step
// is off by the roundings before it, and small singular values suffer most from that; with segments of three and two steps (the
// singular values grow in the first, settle in the second) the result is as exact as step by step, with one of five it would not be.
//
// G, P, T and the products of the Q are symmetric: only the tiles on and above the diagonal are computed, the others are written as
// their transposes.
//
// One 256 x BN tile per two-CTA cluster (tcgen05 cta_group::2), roles as in gemm_pair_sm100.cu:
//   warp 0      TMA producer of this CTA's halves
//   warp 1      MMA issuer (leader CTA only); allocates TMEM in both CTAs
//   warps 2..9  epilogue: accumulator and the tile of G or X that is added to it, which is fetched while the main loop runs
//
// What bounds it: for large matrices the tensor pipe and the power limit (326 us for X = Q X at 4096 x 14336, 1.48 PFLOP/s; products of
// 4096 x 4096 60 us, 1.8 waves of tiles on 74 pairs of SMs), for small ones the chain of launches: 7 us each, of which 1.4 are the
// first load, 1.2 the epilogue and 2.7 the end of one kernel and the start of the next.  One B200, five steps: 2048 x 512 123 us;
// optimizer step 6144 x 4096 1.65 ms, 4096 x 14336 2.48.
#include <cuda_fp16.h>
#include "sm100.cuh"
#include "launch.h"
#include "native_ops.h"
#include "pdl.cuh"
#include "host_utils.h"

namespace kb {

constexpr int NS_BM = 256;                     // rows of a tile (128 per CTA)
constexpr int NS_BK = 64;
constexpr int NS_MAX_STAGES = 8;
constexpr int NS_EPI_WARPS = 8;                // 4 TMEM lane quarters x 2 sets of column slabs
constexpr int NS_THREADS = (2 + NS_EPI_WARPS) * 32;
constexpr int NS_A_BYTES = 128 * NS_BK * 2;
constexpr int NS_RING = 5 * (NS_A_BYTES + 128 * NS_BK * 2);
constexpr int NS_STG_BYTES = NS_EPI_WARPS * 8192;          // two 4 KB slabs a warp
constexpr int NS_SMEM = NS_RING + NS_STG_BYTES + 256 + 1024;
static_assert(NS_SMEM <= 227 * 1024, "shared memory per CTA");

enum NsMode : int {
  NS_GRAM = 0,       // G = X Xt
  NS_POLY = 1,       // P = b G + c G G; diagonal d apart
  NS_UPDATE = 2,     // X <- (a + d) X + P X, or Q X
  NS_UPDATE_T = 3,   // X <- X (a + d) + X P, or X Q
  NS_CARRY = 4,      // Y <- (a + d) Y + P Y for symmetric Y that P commutes with
  NS_GRAM_PARTS = 5, // parts of X Xt along K, as fp32 sums
};
__host__ __device__ constexpr bool ns_symmetric(int mode) { return mode != NS_UPDATE && mode != NS_UPDATE_T; }
__host__ __device__ constexpr bool ns_adds(int mode) { return mode != NS_GRAM && mode != NS_GRAM_PARTS; }

struct NsWork {
  int batch, pairs, tiles_m, tiles_n, per_matrix, nk;      // pairs: matrices per item of the batch (NS_CARRY takes G and Q at once)
  int ratio;                                   // column tiles per 256 rows, where only the upper tiles are computed; else 0
  int group_m;
  int parts;                                   // of the sum over K (NS_GRAM_PARTS): all tiles of part 0, then those of part 1, ...
  __device__ __forceinline__ int tiles() const { return pairs * batch * per_matrix; }
  __device__ __forceinline__ int units() const { return parts * tiles(); }
  __device__ __forceinline__ void steps(int u, int& kb0, int& kb1) const {
    const int part = u / tiles();
    kb0 = split_begin(nk, parts, part);
    kb1 = split_begin(nk, parts, part + 1);
  }
  __device__ __forceinline__ void decode(int u, int& pair, int& z, int& tm, int& tn) const {
    if (parts > 1) u %= tiles();
    z = u / per_matrix;
    int t = u - z * per_matrix;
    pair = z / batch;
    z -= pair * batch;
    if (ratio) {                               // row after row of the upper triangle
      tm = 0;
      for (int len = tiles_n; t >= len; len -= ratio) { t -= len; ++tm; }
      tn = tm * ratio + t;
    } else {
      const int per_group = group_m * tiles_n;
      const int g = t / per_group, first_m = g * group_m, gsz = min(group_m, tiles_m - first_m), r = t - g * per_group;
      tm = first_m + r % gsz;
      tn = r / gsz;
    }
  }
};

struct NsEpilogue {
  const __half* e;           // matrix that is added (G, X or Y): [pairs][batch][M][lde]
  long e_batch, e_pair;
  int lde, e_cols;           // e_cols: columns to read, a multiple of 8
  float alpha, coef;         // accumulator's factor, e's factor
  // Diagonals, [batch][len] each.  `diag`: P's, written by NS_POLY, added to the factor of the row (column) by the updates and
  // NS_CARRY.  e_diag: of the matrix that is added, c_diag: of the result (NS_GRAM, NS_CARRY); from one of a pair to the other diag_pair
  // elements.
  float* diag;
  const float* e_diag;
  float* c_diag;
  long e_diag_pair, c_diag_pair;
  int len;
  float scale[2];            // of the matrix that is added and of the result, for the first and the second of a pair
  float rounded;             // updates by Q: its scale; the factor is what rounding took from the diagonal.  0: updates by P
  float b, c;                // NS_POLY
  float unit;                // 1 / scale of the result
  float also;                // NS_POLY: (a I + P) times this goes to a second matrix, its diagonal to c_diag; 0: not wanted
  float a;
  __nv_bfloat16* out;        // last update: the result, [batch][M][N]
  bool last;
  // last update of an optimizer step: master <- keep * master - step * result, p = bf16(master), of rows of N elements; or null
  float* master;
  __nv_bfloat16* p;
  float keep, step;
};

// One element of that.
__device__ __forceinline__ float muon_weight(float master, float o, float keep, float step) { return fmaf(-step, o, master * keep); }

// What fp16 leaves of v at this scale (a power of two).
__device__ __forceinline__ float rounded16(float v, float scale) { return __half2float(__float2half_rn(v * scale)) / scale; }

// D[tmem] (+)= A * B in fp16: the instruction descriptor's formats are 0.
__host__ __device__ constexpr uint32_t make_idesc_f16(int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void tma_load_4d_pair(void* dst, const CUtensorMap* map, uint32_t cluster_bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(cluster_bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 f16_pair(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// NARROW: tiles of 64 columns, whose epilogue takes slabs of 32 so that both sets of warps have one.
template <bool A_MN, bool B_MN, int MODE, bool NARROW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NS_THREADS, 1)
newton_schulz_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmM,
                     const __grid_constant__ CUtensorMap tmC2, const __grid_constant__ CUtensorMap tmM2, const NsWork w, const int M,
                     const int N, const int bn, const NsEpilogue ep, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + NS_RING + NS_STG_BYTES);   // used in the leader
  uint64_t* empty = full + NS_MAX_STAGES;
  uint64_t* tfull = empty + NS_MAX_STAGES;  // [2]
  uint64_t* tempty = tfull + 2;             // [2] used in the leader
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  const int units = w.units();
  const int half_n = bn >> 1;
  const int b_bytes = B_MN ? ((half_n + 63) / 64) * 64 * NS_BK * 2 : half_n * NS_BK * 2, stage_bytes = NS_A_BYTES + b_bytes;
  const int stages = min(NS_MAX_STAGES, NS_RING / stage_bytes);

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS_MAX_STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2 * NS_EPI_WARPS);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                       // the peer's barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmC);
  }
  pdl_begin();

  if (warp == 0) {
    // ------------------------------------------------------------------ producer (each CTA: its own halves)
    if (elect_one()) {
      const int b_chunks = (half_n + 63) >> 6;
      const uint32_t full0 = cluster_addr(full, 0);
      int s = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (int u = first; u < units && ok; u += step) {
        int pair, z, tm, tn;
        w.decode(u, pair, z, tm, tn);
        const int pa = MODE == NS_CARRY ? 0 : pair;      // P serves both
        int kb0 = 0, kb1 = w.nk;
        if constexpr (MODE == NS_GRAM_PARTS) w.steps(u, kb0, kb1);
        const int m0 = tm * NS_BM + rank * 128, n0 = tn * bn + rank * half_n;
        for (int kb_ = kb0; kb_ < kb1; ++kb_) {
          if (!mbar_wait(&empty[s], ph, abort_flag, status, ST_TIMEOUT_EMPTY)) { ok = false; break; }
          uint8_t* a_dst = smem + s * stage_bytes;
          uint8_t* b_dst = a_dst + NS_A_BYTES;
          const uint32_t bar = full0 + s * 8;
          if (rank == 0) mbar_expect_tx(&full[s], 2u * stage_bytes);
          const int k0 = kb_ * NS_BK;
          if constexpr (!A_MN) {
            tma_load_4d_pair(a_dst, &tmA, bar, k0, m0, z, pa);
          } else {
            tma_load_4d_pair(a_dst, &tmA, bar, m0, k0, z, pa);
            tma_load_4d_pair(a_dst + 8192, &tmA, bar, m0 + 64, k0, z, pa);
          }
          if constexpr (!B_MN) {
            tma_load_4d_pair(b_dst, &tmB, bar, k0, n0, z, pair);
          } else {
            tma_load_4d_pair(b_dst, &tmB, bar, n0, k0, z, pair);
            if (b_chunks > 1) tma_load_4d_pair(b_dst + 8192, &tmB, bar, n0 + 64, k0, z, pair);
          }
          if (++s == stages) { s = 0; ph ^= 1u; }
        }
      }
      if (!ok) {
        // leave no copy in flight: tile loads land within microseconds, give them 200 us
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) {}
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (leader)
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = make_idesc_f16(NS_BM, bn, A_MN, B_MN);
      const uint32_t smem0 = smem_u32(smem);
      const uint64_t ad0 = A_MN ? make_smem_desc(smem0, 8192, 1024) : make_smem_desc(smem0, 16, 1024);
      const uint64_t bd0 = B_MN ? make_smem_desc(smem0 + NS_A_BYTES, 8192, 1024) : make_smem_desc(smem0 + NS_A_BYTES, 16, 1024);
      constexpr uint64_t ka = (A_MN ? 2048 : 32) >> 4, kb = (B_MN ? 2048 : 32) >> 4;   // descriptor step of 16 in K
      uint32_t tile_i = 0;
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int u = first; u < units && ok; u += step, ++tile_i) {
        const uint32_t buf = tile_i & 1u;
        if (!mbar_wait(&tempty[buf], ((tile_i >> 1) & 1u) ^ 1u, abort_flag, status, ST_TIMEOUT_TMEM_EMPTY)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * 256;
        int kb0 = 0, kb1 = w.nk;
        if constexpr (MODE == NS_GRAM_PARTS) w.steps(u, kb0, kb1);
        for (int kb_ = kb0; kb_ < kb1; ++kb_) {
          if (!mbar_wait(&full[s], ph, abort_flag, status, ST_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint64_t ad = ad0 + static_cast<uint64_t>(s * (stage_bytes >> 4));
          const uint64_t bd = bd0 + static_cast<uint64_t>(s * (stage_bytes >> 4));
#pragma unroll
          for (int k = 0; k < NS_BK / 16; ++k)
            umma_ss_pair(d_tmem, ad + k * ka, bd + k * kb, idesc, (kb_ > kb0 || k > 0) ? 1u : 0u);
          umma_commit_pair(&empty[s]);
          if (kb_ == kb1 - 1) umma_commit_pair(&tfull[buf]);
          if (++s == stages) { s = 0; ph ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3;                   // TMEM lane quarter
    const int h = (warp - 2) >> 2;            // this warp takes the column slabs h, h + 2, ...
    constexpr int HALVES = NARROW ? 1 : 2;    // of 32 columns in a slab
    constexpr int SLAB = 32 * HALVES, UNITS = SLAB / 8, ROW = UNITS * 16;      // columns, 16-byte units and bytes of a slab's row
    // units are swizzled by row, as TMA expects rows of 64 or 128 bytes
    const auto swizzle = [](int r) { return NARROW ? (r >> 1) & 3 : r & 7; };
    uint8_t* const stg0 = smem + NS_RING + (warp - 2) * 8192;
    const int slabs = bn / SLAB;              // at least two, one for either set of warps
    constexpr bool ADDS = ns_adds(MODE), SYMMETRIC = ns_symmetric(MODE);
    uint4 v[UNITS];                           // the slab that is added, on its way
    float2 d_next = make_float2(0.f, 0.f);    // NS_UPDATE_T: P's diagonal for two of these columns, lane by lane
    auto fetch = [&](int u, int c) {
      int pair, z, tm, tn;
      w.decode(u, pair, z, tm, tn);
      const int row0 = tm * NS_BM + rank * 128 + q * 32, col = tn * bn + c * SLAB + lane % UNITS * 8;
      const __half* src = ep.e + pair * ep.e_pair + z * ep.e_batch + col;
#pragma unroll
      for (int i = 0; i < UNITS; ++i) {
        const int r = row0 + i * (32 / UNITS) + lane / UNITS;
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < M && col < ep.e_cols) v[i] = *reinterpret_cast<const uint4*>(src + static_cast<size_t>(r) * ep.lde);
      }
      if constexpr (MODE == NS_UPDATE_T) {
        const int dc = tn * bn + c * SLAB + 2 * lane;
        const float* d = ep.diag + static_cast<size_t>(z) * ep.len;
        d_next = make_float2(dc < N ? d[dc] : 0.f, dc + 1 < N ? d[dc + 1] : 0.f);
        if (ep.rounded != 0.f) {
          d_next.x -= rounded16(d_next.x, ep.rounded);
          d_next.y -= rounded16(d_next.y, ep.rounded);
        }
      }
    };
    if (ADDS && first < units) fetch(first, h);
    uint32_t tile_i = 0, slab_i = 0;
    for (int u = first; u < units; u += step, ++tile_i) {
      int pair, z, tm, tn;
      w.decode(u, pair, z, tm, tn);
      const uint32_t buf = tile_i & 1u;
      const int row0 = tm * NS_BM + rank * 128 + q * 32, row = row0 + lane;
      float coef = ep.coef;
      float correction = 0.f;                 // of this row's diagonal element, for what rounding took from those that it is made of
      {
        const size_t at = static_cast<size_t>(z) * ep.len + row;
        if constexpr (MODE == NS_UPDATE || MODE == NS_CARRY) {
          if (row < M) {
            const float d = ep.diag[at];
            coef += MODE == NS_UPDATE && ep.rounded != 0.f ? d - rounded16(d, ep.rounded) : d;
          }
        }
        if constexpr (MODE == NS_CARRY || MODE == NS_POLY) {
          if (row < M) {
            const float scale = ep.scale[pair], v = ep.e_diag[pair * ep.e_diag_pair + at], lost = v - rounded16(v, scale);
            correction = MODE == NS_CARRY ? coef * lost * scale : (ep.b * lost + ep.c * lost * (2.f * v - lost)) * scale;
          }
        }
      }
      __syncwarp();
      if (!mbar_wait_warp(&tfull[buf], (tile_i >> 1) & 1u, abort_flag, status, ST_TIMEOUT_TMEM_FULL)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + buf * 256 + (static_cast<uint32_t>(q * 32) << 16);
      const bool reused = u + 2 * step < units;      // a later tile takes this accumulator; handing it back costs half a microsecond
      const bool mirror = SYMMETRIC && tn * bn / NS_BM > tm;
#pragma unroll 1
      for (int c = h; c < slabs; c += 2, ++slab_i) {
        // Symmetric outputs use one buffer for the tile and one for its transpose, the others two in turn.
        uint8_t* const stg = SYMMETRIC ? stg0 : stg0 + (slab_i & 1u) * 4096;
        uint8_t* const stg_row = stg + lane * ROW;
        const float2 d_now = d_next;
        if (lane == 0) {
          if constexpr (SYMMETRIC) tma_store_wait_read<0>();
          else tma_store_wait_read<1>();
        }
        __syncwarp();
        if constexpr (ADDS) {
#pragma unroll
          for (int i = 0; i < UNITS; ++i) {
            const int r = i * (32 / UNITS) + lane / UNITS;
            *reinterpret_cast<uint4*>(stg + r * ROW + ((lane % UNITS ^ swizzle(r)) << 4)) = v[i];
          }
          __syncwarp();
          if (c + 2 < slabs) fetch(u, c + 2);
          else if (u + step < units) fetch(u + step, h);
          __syncwarp();
        }
        const int col0 = tn * bn + c * SLAB;
        if constexpr (MODE == NS_GRAM_PARTS) {           // the sums themselves, 32 columns at a time, to the workspace
#pragma unroll
          for (int half = 0; half < HALVES; ++half) {
            uint32_t a[32];
            __syncwarp();
            tmem_ld_32x32(taddr + c * SLAB + half * 32, a);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 8; ++j)
              st_shared_v4(smem_u32(stg0) + lane * 128 + half * 4096 + ((j ^ (lane & 7)) << 4), a[4 * j], a[4 * j + 1], a[4 * j + 2],
                           a[4 * j + 3]);
          }
          if (c + 2 >= slabs) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && reused) mbar_arrive_cluster(cluster_addr(&tempty[buf], 0));
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            for (int half = 0; half < HALVES; ++half)
              tma_store_2d(&tmC2, stg0 + half * 4096, c * SLAB + half * 32, u * NS_BM + rank * 128 + q * 32);
            tma_store_commit();
          }
          continue;
        }
        uint32_t o[16 * HALVES];
        uint32_t o2[MODE == NS_POLY ? 16 * HALVES : 1];  // a I + P
        // the diagonal crosses few slabs: the others are spared the search for it
        const bool on_diagonal = SYMMETRIC && col0 < row0 + 32 && row0 < col0 + SLAB;
        float diagonal = 0.f;
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          uint32_t a[32];
          float f[32];
          __syncwarp();                               // TMEM is read by whole warps: what lanes did on their own before ends here
          tmem_ld_32x32(taddr + c * SLAB + half * 32, a);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int unit = half * 4 + j;
            uint4 e4 = make_uint4(0u, 0u, 0u, 0u);
            if constexpr (ADDS) e4 = *reinterpret_cast<const uint4*>(stg_row + ((unit ^ swizzle(lane)) << 4));
            const uint32_t e[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int k = 8 * j + 2 * i;
              float x = __uint_as_float(a[k]) * ep.alpha, y = __uint_as_float(a[k + 1]) * ep.alpha;
              if constexpr (ADDS) {
                const float2 p = f16_pair(e[i]);
                float c0 = coef, c1 = coef;
                if constexpr (MODE == NS_UPDATE_T) {
                  c0 += __shfl_sync(0xffffffffu, d_now.x, half * 16 + k / 2);
                  c1 += __shfl_sync(0xffffffffu, d_now.y, half * 16 + k / 2);
                }
                x = fmaf(c0, p.x, x);
                y = fmaf(c1, p.y, y);
              }
              f[k] = x;
              f[k + 1] = y;
            }
          }
          if constexpr (MODE == NS_POLY) {
            if (ep.also != 0.f) {
#pragma unroll
              for (int i = 0; i < 16; ++i) o2[half * 16 + i] = pack_f16x2(f[2 * i] * ep.also, f[2 * i + 1] * ep.also);
            }
          }
          if (on_diagonal) {
            const int at = row - col0 - half * 32;        // this row's diagonal element, if it is here
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const bool d0 = at == 2 * i, d1 = at == 2 * i + 1;
              diagonal = d0 ? f[2 * i] + correction : d1 ? f[2 * i + 1] + correction : diagonal;
              if constexpr (MODE == NS_POLY) {
                if (ep.also != 0.f && (d0 || d1)) {
                  const float whole = (diagonal * ep.unit + ep.a) * (ep.also / ep.unit);
                  o2[half * 16 + i] = d0 ? pack_f16x2(whole, f[2 * i + 1] * ep.also) : pack_f16x2(f[2 * i] * ep.also, whole);
                }
                f[2 * i] = d0 ? 0.f : f[2 * i];
                f[2 * i + 1] = d1 ? 0.f : f[2 * i + 1];
              } else {
                f[2 * i] = d0 ? diagonal : f[2 * i];
                f[2 * i + 1] = d1 ? diagonal : f[2 * i + 1];
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 16; ++i)
            o[half * 16 + i] = ep.last ? pack_bf16x2(f[2 * i] * ep.unit, f[2 * i + 1] * ep.unit) : pack_f16x2(f[2 * i], f[2 * i + 1]);
        }
        if (on_diagonal && row >= col0 && row < col0 + SLAB && row < M) {
          const size_t at = static_cast<size_t>(z) * ep.len + row;
          if constexpr (MODE == NS_POLY) {
            ep.diag[at] = diagonal * ep.unit;
            if (ep.also != 0.f) ep.c_diag[at] = diagonal * ep.unit + ep.a;
          } else {
            ep.c_diag[pair * ep.c_diag_pair + at] = diagonal / ep.scale[pair];
          }
        }
        if (c + 2 >= slabs) {
          // this warp's last read of the accumulator: hand it back before the stores go out
          tc_fence_before();
          __syncwarp();
          if (lane == 0 && reused) mbar_arrive_cluster(cluster_addr(&tempty[buf], 0));
        }
        __syncwarp();
        if (!SYMMETRIC && ep.last && (N & 7)) {      // rows of the result start anywhere
          __nv_bfloat16* dst = ep.out + (static_cast<size_t>(z) * M + row) * N + col0;
          if (row < M) {
#pragma unroll
            for (int j = 0; j < SLAB; ++j)
              if (col0 + j < N) dst[j] = __ushort_as_bfloat16(static_cast<unsigned short>(o[j >> 1] >> (j & 1 ? 16 : 0)));
          }
          continue;
        }
        const bool here = row0 < M && col0 < N;      // the tensor maps clip what crosses the edge
        auto put = [&](const uint32_t* v, const CUtensorMap* direct, const CUtensorMap* transposed) {
#pragma unroll
          for (int j = 0; j < UNITS; ++j)
            st_shared_v4(smem_u32(stg_row) + ((j ^ swizzle(lane)) << 4), v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          if (mirror) {                              // [columns][32 rows]
            uint16_t* t = reinterpret_cast<uint16_t*>(stg0 + 4096) + lane;
#pragma unroll
            for (int j = 0; j < 16 * HALVES; ++j) {
              t[(2 * j) * 32] = static_cast<uint16_t>(v[j]);
              t[(2 * j + 1) * 32] = static_cast<uint16_t>(v[j] >> 16);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (here) {
              tma_store_4d(direct, stg, col0, row0, z, pair);
              if (mirror) tma_store_4d(transposed, stg0 + 4096, row0, col0, z, pair);
            }
            tma_store_commit();
          }
        };
        put(o, &tmC, &tmM);
        if constexpr (!SYMMETRIC) {
          if (ep.master) {                           // eight columns a lane, from the slab that is being stored
#pragma unroll 4
            for (int i = 0; i < UNITS; ++i) {
              const int r = i * (32 / UNITS) + lane / UNITS, u8 = lane % UNITS;
              if (row0 + r >= M || col0 + u8 * 8 >= N) continue;
              const uint4 x = *reinterpret_cast<const uint4*>(stg + r * ROW + ((u8 ^ swizzle(r)) << 4));
              const size_t at = static_cast<size_t>(row0 + r) * N + col0 + u8 * 8;
              float4* m = reinterpret_cast<float4*>(ep.master + at);
              float4 a = m[0], b = m[1];
              a.x = muon_weight(a.x, __uint_as_float(x.x << 16), ep.keep, ep.step);
              a.y = muon_weight(a.y, __uint_as_float(x.x & 0xffff0000u), ep.keep, ep.step);
              a.z = muon_weight(a.z, __uint_as_float(x.y << 16), ep.keep, ep.step);
              a.w = muon_weight(a.w, __uint_as_float(x.y & 0xffff0000u), ep.keep, ep.step);
              b.x = muon_weight(b.x, __uint_as_float(x.z << 16), ep.keep, ep.step);
              b.y = muon_weight(b.y, __uint_as_float(x.z & 0xffff0000u), ep.keep, ep.step);
              b.z = muon_weight(b.z, __uint_as_float(x.w << 16), ep.keep, ep.step);
              b.w = muon_weight(b.w, __uint_as_float(x.w & 0xffff0000u), ep.keep, ep.step);
              m[0] = a;
              m[1] = b;
              *reinterpret_cast<uint4*>(ep.p + at) =
                  make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w));
            }
            __syncwarp();
          }
        }
        if constexpr (MODE == NS_POLY) {
          if (ep.also != 0.f) {
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
            put(o2, &tmC2, &tmM2);
          }
        }
      }
    }
    if (lane == 0) tma_store_wait_read<0>();         // nothing in flight out of shared memory at exit
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// G from the sums of its parts along K, added in order: 32 x 32 elements a block, as they are and transposed.
__global__ void __launch_bounds__(256)
ns_sum_parts_kernel(const float* __restrict__ work, __half* __restrict__ G, long ldg, int side, int bn, const NsWork w, float alpha,
                    float* __restrict__ diag) {
  __shared__ float t[32][33];
  pdl_begin();
  const int per_tile = 8 * (bn / 32), tile = blockIdx.x / per_tile, sub = blockIdx.x - tile * per_tile;
  int pair, z, tm, tn;
  w.decode(tile, pair, z, tm, tn);
  const int r0 = sub % 8 * 32, c0 = sub / 8 * 32;       // inside the tile
  const int row0 = tm * NS_BM + r0, col0 = tn * bn + c0;
  if (row0 >= side || col0 >= side) return;
  const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 4;
  const float* src = work + (static_cast<size_t>(tile) * NS_BM + r0 + r) * bn + c0 + c;
  const size_t part = static_cast<size_t>(w.tiles()) * NS_BM * bn;
  float4 s = *reinterpret_cast<const float4*>(src);
#pragma unroll 4
  for (int p = 1; p < w.parts; ++p) {
    const float4 x = *reinterpret_cast<const float4*>(src + p * part);
    s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
  }
  s.x *= alpha; s.y *= alpha; s.z *= alpha; s.w *= alpha;
  const int on = row0 + r - col0 - c;                   // which of the four columns the row's diagonal element is in
  if (on >= 0 && on < 4 && row0 + r < side)
    diag[static_cast<size_t>(z) * side + row0 + r] = (on == 0 ? s.x : on == 1 ? s.y : on == 2 ? s.z : s.w) * alpha;
  __half* g = G + static_cast<size_t>(z) * side * ldg;
  // rows hold whole groups of eight columns; what lies behind the last column is zero
  if (row0 + r < side && col0 + c < ldg)
    *reinterpret_cast<uint2*>(g + (row0 + r) * ldg + col0 + c) = make_uint2(pack_f16x2(s.x, s.y), pack_f16x2(s.z, s.w));
  if (tn * bn / NS_BM == tm) return;
  t[r][c] = s.x; t[r][c + 1] = s.y; t[r][c + 2] = s.z; t[r][c + 3] = s.w;
  __syncthreads();
  if (col0 + r < side && row0 + c < ldg)
    *reinterpret_cast<uint2*>(g + (col0 + r) * ldg + row0 + c) =
        make_uint2(pack_f16x2(t[c][r], t[c + 1][r]), pack_f16x2(t[c + 2][r], t[c + 3][r]));
}

// ----------------------------------------------------------------------------- the passes around the products
constexpr int NS_SUM_THREADS = 256;
constexpr int NS_SUM_BLOCKS = 592;             // most blocks that share a matrix' sum of squares

__device__ __forceinline__ double block_sum(double s) {
  __shared__ double sh[NS_SUM_THREADS / 32];
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.;
#pragma unroll
  for (int i = 0; i < NS_SUM_THREADS / 32; ++i) s += sh[i];
  return s;
}

// The matrix that is orthogonalised, read where it lies: of fp32 or bf16 values, or of a gradient and its momentum.
struct NsSource {
  const void* x;             // fp32 or bf16 values; the gradient of an optimizer step
  float* m;                  // momentum, or null
  const float* grad_scale;   // the gradient's factor on the device, or null
  float beta;
  bool bf16, nesterov;
  // eight values from element `at` on (`n` of them exist), `whole`: aligned and all there
  template <bool STEP>
  __device__ __forceinline__ void load(long at, int n, bool whole, float gs, float (&u)[8]) const {
    float g[8];
    if (bf16) {
      const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(x) + at;
      if (whole) {
        const uint4 r = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          g[2 * j] = __uint_as_float(w[j] << 16);
          g[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = j < n ? __bfloat162float(p[j]) : 0.f;
      }
    } else {
      load8(static_cast<const float*>(x) + at, n, whole, g);
    }
    if (!m) {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = g[j];
      return;
    }
    float mo[8];
    load8(m + at, n, whole, mo);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      g[j] *= gs;
      if (STEP) mo[j] = fmaf(beta, mo[j], g[j]);
      u[j] = nesterov ? fmaf(beta, mo[j], g[j]) : mo[j];
    }
    if (STEP) {
      if (whole) {
        *reinterpret_cast<float4*>(m + at) = make_float4(mo[0], mo[1], mo[2], mo[3]);
        *reinterpret_cast<float4*>(m + at + 4) = make_float4(mo[4], mo[5], mo[6], mo[7]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < n) m[at + j] = mo[j];
      }
    }
  }
  static __device__ __forceinline__ void load8(const float* p, int n, bool whole, float (&g)[8]) {
    if (whole) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      g[0] = a.x; g[1] = a.y; g[2] = a.z; g[3] = a.w;
      g[4] = b.x; g[5] = b.y; g[6] = b.z; g[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = j < n ? p[j] : 0.f;
    }
  }
};

// Momentum step (where there is one) and sum of squares: part[matrix][block], in a fixed order.
__global__ void __launch_bounds__(NS_SUM_THREADS)
ns_sumsq_kernel(const NsSource src, long count, bool aligned, double* __restrict__ part) {
  pdl_begin();
  const float gs = src.grad_scale ? *src.grad_scale : 1.f;
  const long base = blockIdx.y * count, vecs = (count + 7) / 8;
  float s = 0.f;
  double total = 0.;
  int n = 0;
  for (long i = static_cast<long>(blockIdx.x) * NS_SUM_THREADS + threadIdx.x; i < vecs; i += static_cast<long>(gridDim.x) * NS_SUM_THREADS) {
    const int left = static_cast<int>(count - i * 8 < 8 ? count - i * 8 : 8);
    float u[8];
    src.load<true>(base + i * 8, left, aligned && left == 8, gs, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(u[j], u[j], s);
    if (++n == 32) {                           // short fp32 sums, added up in fp64
      total += s;
      s = 0.f;
      n = 0;
    }
  }
  total = block_sum(total + s);
  if (threadIdx.x == 0) part[static_cast<size_t>(blockIdx.y) * gridDim.x + blockIdx.x] = total;
}

// X_0 in fp16: rows of ldx elements, zeros behind the columns.
__global__ void __launch_bounds__(NS_SUM_THREADS)
ns_normalize_kernel(const NsSource src, int rows, int cols, int ldx, bool aligned, const double* __restrict__ part, int parts, float eps,
                    float scale, __half* __restrict__ x) {
  pdl_begin();
  double sq = 0.;
  for (int i = threadIdx.x; i < parts; i += NS_SUM_THREADS) sq += part[static_cast<size_t>(blockIdx.y) * parts + i];
  const double norm = sqrt(block_sum(sq)) + static_cast<double>(eps);
  // a norm that fp32 squares cannot hold, or a matrix with an infinity, gives NaN and not zeros
  const float f = isinf(norm) ? __int_as_float(0x7fc00000) : static_cast<float>(static_cast<double>(scale) / norm);
  const float gs = src.grad_scale ? *src.grad_scale : 1.f;
  const int vecs = ldx >> 3;
  const long total = static_cast<long>(rows) * vecs;
  const long base = blockIdx.y * static_cast<long>(rows) * cols;
  x += blockIdx.y * static_cast<long>(rows) * ldx;
  for (long i = static_cast<long>(blockIdx.x) * NS_SUM_THREADS + threadIdx.x; i < total; i += static_cast<long>(gridDim.x) * NS_SUM_THREADS) {
    const long r = i / vecs;
    const int c = static_cast<int>(i - r * vecs) * 8, left = min(8, cols - c);
    float u[8];
    src.load<false>(base + r * cols + c, left, aligned && left == 8, gs, u);
    uint4 o;
    o.x = pack_f16x2(u[0] * f, u[1] * f);
    o.y = pack_f16x2(u[2] * f, u[3] * f);
    o.z = pack_f16x2(u[4] * f, u[5] * f);
    o.w = pack_f16x2(u[6] * f, u[7] * f);
    *reinterpret_cast<uint4*>(x + i * 8) = o;
  }
}

// The same where rows of the result start anywhere, so that the product's epilogue cannot take it along.
__global__ void __launch_bounds__(256)
muon_apply_kernel(float* __restrict__ master, __nv_bfloat16* __restrict__ p, const __nv_bfloat16* __restrict__ o, long n, float keep,
                  float step) {
  pdl_begin();
  for (long i = static_cast<long>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<long>(gridDim.x) * 256) {
    const float a = muon_weight(master[i], __bfloat162float(o[i]), keep, step);
    master[i] = a;
    p[i] = __float2bfloat16(a);
  }
}

// ----------------------------------------------------------------------------- host side
constexpr int NS_G = 0, NS_T = 1, NS_Q = 2, NS_P = 4, NS_SLOTS = 5;      // square matrices of the workspace: G, T, two Q, P

// How a product is cut: tile width, tiles and parts of the sum over K.
struct NsPlan {
  int bn, tiles_m, tiles_n, per_matrix, nk, parts;
  double clocks;             // modelled time, with 6 to 7 us for a launch, its first loads and its epilogue, 5 us for adding up parts
};
static NsPlan ns_plan(int mode, long matrices, int M, int N, int K) {
  const bool symmetric = ns_symmetric(mode);
  const int sms = device_sm_count() / 2;
  NsPlan p{};
  p.tiles_m = (M + NS_BM - 1) / NS_BM;
  p.nk = (K + NS_BK - 1) / NS_BK;
  p.parts = 1;
  // Width of the tiles: as for the other products on pairs of SMs, clocks of a step of 64 are the larger of the tensor cores' (2 a
  // column) and of the loads' (64 bytes a clock reach an SM).
  double best = 0, step = 0;
  for (int b = 256; b >= 64; b -= 64) {
    if (symmetric && 256 % b) continue;        // rows of tiles start on the diagonal
    const int tn = (N + b - 1) / b;
    long tiles = 0;
    if (symmetric) for (int i = 0; i < p.tiles_m; ++i) tiles += tn - i * (256 / b);
    else tiles = (long)p.tiles_m * tn;
    const long waves = (tiles * matrices + sms - 1) / sms;
    const double clocks = 2 * b > 256 + b ? 2 * b : 256 + b, cost = (double)waves * (p.nk * clocks + 1500.0);
    if (!p.bn || cost < best * 0.97) {
      best = cost;
      step = clocks;
      p.bn = b;
      p.tiles_n = tn;
      p.per_matrix = (int)tiles;
    }
  }
  // Few tiles and a long sum: parts of 8 steps and more on the SMs that would idle, where that saves more than the 5 us that adding
  // them up takes.  20 x 14336, step by step: 316 us as one part, 134 so.
  if (mode == NS_GRAM) {
    const long units = matrices * p.per_matrix;
    long parts = units ? sms / units : 1;
    parts = parts > p.nk / 8 ? p.nk / 8 : parts;
    if (parts > 1 && (p.nk - (p.nk + parts - 1) / parts) * step > 10000.) {
      p.parts = (int)parts;
      best = (p.nk + parts - 1) / parts * step + 1500. + 10000.;
    }
  }
  p.clocks = best + (mode == NS_CARRY ? 11000. : 13000.);
  return p;
}

struct NsLayout {
  int rows, cols, side;      // side: the smaller of the two
  long ldx, ldg;             // row strides in elements (multiples of 8)
  long x, g, diag, part, sums, total;          // bytes; g: one square matrix of every item; sums: parts of a G
  NsLayout(int batch, int m, int n) : rows(m), cols(n), side(m < n ? m : n) {
    const auto up = [](long b) { return (b + 255) / 256 * 256; };
    ldx = (n + 7L) / 8 * 8;
    ldg = (side + 7L) / 8 * 8;
    x = up(2L * batch * m * ldx);
    g = up(2L * batch * side * ldg);
    diag = up(4L * NS_SLOTS * batch * side);
    part = up(8L * batch * NS_SUM_BLOCKS);
    const NsPlan p = ns_plan(NS_GRAM, batch, side, side, m < n ? n : m);
    sums = p.parts > 1 ? up(4L * p.parts * batch * p.per_matrix * NS_BM * p.bn) : 0;
    total = 2 * x + NS_SLOTS * g + diag + part + sums;
  }
};

// Matrices of one product: [pairs][batch][rows][ld]; pair_bytes: from the first of a pair to the second.
struct NsMatrix {
  void* p;
  long ld;
  long pair_bytes;
};

static int ns_map(CUtensorMap* map, const NsMatrix& m, long inner, long rows, long batch, int pairs, uint32_t box_inner, uint32_t box_rows,
                  int swizzle) {
  const uint64_t item = (uint64_t)m.ld * rows * 2;
  const uint64_t dims[4] = {(uint64_t)inner, (uint64_t)rows, (uint64_t)batch, (uint64_t)pairs};
  const uint64_t str[3] = {(uint64_t)m.ld * 2, item, pairs > 1 ? (uint64_t)m.pair_bytes : item * batch};
  const uint32_t box[4] = {box_inner, box_rows, 1, 1};
  return make_tmap(map, m.p, 2, 4, dims, str, box, swizzle);
}

// C [M, N] of each matrix of the batch from A and B: [rows][ld] matrices whose rows run along K (K-major) or along M / N.
template <bool A_MN, bool B_MN, int MODE>
static int ns_product(const NsMatrix& A, const NsMatrix& B, const NsMatrix& C, const NsMatrix& C2, int batch, int pairs, int M, int N, int K,
                      const NsEpilogue& ep, float* sums, int* status, cudaStream_t stream) {
  constexpr bool SYMMETRIC = ns_symmetric(MODE);
  const int sms = device_sm_count() / 2;
  const NsPlan plan = ns_plan(MODE, (long)batch * pairs, M, N, K);
  const int bn = plan.bn;
  NsWork w;
  w.batch = batch;
  w.pairs = pairs;
  w.tiles_m = plan.tiles_m;
  w.tiles_n = plan.tiles_n;
  w.per_matrix = plan.per_matrix;
  w.nk = plan.nk;
  w.parts = plan.parts;
  w.ratio = SYMMETRIC ? 256 / bn : 0;
  long gm = (24L << 20) / ((long)NS_BM * K * 2);
  gm = gm < 8 ? 8 : gm > 16 ? 16 : gm;
  w.group_m = gm < w.tiles_m ? (int)gm : w.tiles_m;
  CUtensorMap tmA, tmB, tmC, tmM, tmC2, tmM2;
  int rc;
  const int pairs_a = MODE == NS_CARRY ? 1 : pairs;
  // operands: zeros past the edge of K and of the rows, so that padding never counts
  if (!A_MN) rc = ns_map(&tmA, A, K, M, batch, pairs_a, NS_BK, 128, 3);
  else       rc = ns_map(&tmA, A, M, K, batch, pairs_a, 64, NS_BK, 3);
  if (rc) return rc;
  if (!B_MN) rc = ns_map(&tmB, B, K, N, batch, pairs, NS_BK, bn / 2, 3);
  else       rc = ns_map(&tmB, B, N, K, batch, pairs, 64, NS_BK, 3);
  if (rc) return rc;
  // the output's rows in whole 16-byte units (the padding of the workspace takes zeros); a result with other rows is not stored by TMA
  tmC = tmA;
  const bool narrow = bn == 64;                // the others have 128 columns and more: two slabs a tile at least in either form
  const uint32_t slab = narrow ? 32 : 64;
  const int swizzle = narrow ? 2 : 3;
  if (C.ld % 8 == 0 && (rc = ns_map(&tmC, C, C.ld, M, batch, pairs, slab, 32, swizzle))) return rc;
  tmM = tmC;
  if (SYMMETRIC && (rc = ns_map(&tmM, C, C.ld, M, batch, pairs, 32, slab, 0))) return rc;
  tmC2 = tmC;
  tmM2 = tmM;
  if (MODE == NS_POLY && C2.p && ((rc = ns_map(&tmC2, C2, C2.ld, M, batch, pairs, slab, 32, swizzle)) ||
                                  (rc = ns_map(&tmM2, C2, C2.ld, M, batch, pairs, 32, slab, 0))))
    return rc;
  const long units = (long)plan.parts * pairs * batch * w.per_matrix;
  if (units >= 1L << 22) return 7;
  if (MODE == NS_GRAM && plan.parts > 1) {
    const uint64_t dims[2] = {(uint64_t)bn, (uint64_t)units * NS_BM}, str[1] = {(uint64_t)bn * 4};
    const uint32_t box[2] = {32u, 32u};
    if ((rc = make_tmap(&tmC2, sums, 4, 2, dims, str, box, 3))) return rc;
  }
  constexpr int PARTS = MODE == NS_GRAM ? NS_GRAM_PARTS : MODE;
  auto kern = plan.parts > 1 ? (narrow ? newton_schulz_kernel<A_MN, B_MN, PARTS, true> : newton_schulz_kernel<A_MN, B_MN, PARTS, false>)
                             : (narrow ? newton_schulz_kernel<A_MN, B_MN, MODE, true> : newton_schulz_kernel<A_MN, B_MN, MODE, false>);
  const int variant = (plan.parts > 1 ? 2 : 0) + (narrow ? 1 : 0);
  static bool configured[4][64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 7;
  if (!configured[variant][dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM);
    if (e != cudaSuccess) return 1000 + static_cast<int>(e);
    configured[variant][dev] = true;
  }
  const int grid = 2 * (int)(units < sms ? units : sms);
  KB_LAUNCH_PDL(kern, grid, NS_THREADS, NS_SMEM, stream, tmA, tmB, tmC, tmM, tmC2, tmM2, w, M, N, bn, ep, status);
  if (MODE == NS_GRAM && plan.parts > 1)
    KB_LAUNCH_PDL(ns_sum_parts_kernel, (unsigned)(batch * w.per_matrix * 8 * (bn / 32)), 256, 0, stream, (const float*)sums,
                  static_cast<__half*>(C.p), C.ld, M, bn, w, ep.alpha, ep.c_diag);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 2000 + static_cast<int>(e);
}

// Whether G is carried from step to step (see the head of this file): where the longer side is at least 1.5 times the other and the
// modelled time is less.  One B200, us step by step / carried: 14336 x 4096 3650 / 2560, 6144 x 4096 1842 / 1675, 1024 x 4096 195 / 177,
// 20 x 14336 134 / 109; where all products are over before their launches and epilogues are there is nothing to gain: 2048 x 512 139 /
// 143, three of 333 x 1000 126 / 138.
static bool ns_carries(int batch, int m, int n, int steps) {
  const int side = m < n ? m : n, other = m < n ? n : m;
  if (steps < 2 || 2L * other < 3L * side) return false;
  const bool tall = m > n;
  const double gram = ns_plan(NS_GRAM, batch, side, side, other).clocks, square = ns_plan(NS_CARRY, batch, side, side, side).clocks;
  const double x = ns_plan(NS_UPDATE, batch, tall ? other : side, tall ? side : other, side).clocks;
  const int segments = steps / 2, products = 3 * steps - segments + steps % 2;    // of G's size: P, T, G' and products of Q
  return segments * (gram + x) + products * square < steps * (gram + square + x);
}
// Steps of the segment that begins with `left` steps to go: three and then two, or only two.
static int ns_segment(bool carries, int left) {
  if (!carries) return 1;
  return left % 2 == 1 && left > 1 ? 3 : left < 2 ? left : 2;
}

// What the last product of an optimizer step does beside its result.
struct MuonApply {
  float* master;
  __nv_bfloat16* p;
  float keep, step;
};

static int newton_schulz(const NsSource& src, const MuonApply& apply, int batch, int m, int n, float a, float b, float c, int steps,
                         float eps, float scale, float scale_q, void* out, uint8_t* work, int* status, cudaStream_t stream) {
  const NsLayout lay(batch, m, n);
  uint8_t* const x[2] = {work, work + lay.x};
  uint8_t* const square = work + 2 * lay.x;
  float* const diag = reinterpret_cast<float*>(square + NS_SLOTS * lay.g);
  double* const part = reinterpret_cast<double*>(square + NS_SLOTS * lay.g + lay.diag);
  float* const sums = reinterpret_cast<float*>(square + NS_SLOTS * lay.g + lay.diag + lay.part);
  const long count = (long)m * n;
  const auto al = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  const long per_block = 8L * NS_SUM_THREADS;
  {
    const bool aligned = al(src.x) && al(src.m) && (batch == 1 || count % 8 == 0);
    long blocks = (count + 4 * per_block - 1) / (4 * per_block);
    const long most = NS_SUM_BLOCKS / batch > 1 ? NS_SUM_BLOCKS / batch : 1;
    blocks = blocks < 1 ? 1 : blocks > most ? most : blocks;
    KB_LAUNCH_PDL(ns_sumsq_kernel, dim3((unsigned)blocks, batch), NS_SUM_THREADS, 0, stream, src, count, aligned, part);
    const bool rows_aligned = al(src.x) && al(src.m) && n % 8 == 0;
    long nblocks = (m * (lay.ldx / 8) + NS_SUM_THREADS - 1) / NS_SUM_THREADS;
    nblocks = nblocks > 148 * 8 ? 148 * 8 : nblocks;
    KB_LAUNCH_PDL(ns_normalize_kernel, dim3((unsigned)nblocks, batch), NS_SUM_THREADS, 0, stream, src, m, n, (int)lay.ldx, rows_aligned,
                  (const double*)part, (int)blocks, eps, scale, reinterpret_cast<__half*>(x[0]));
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return 2000 + static_cast<int>(e);
  }
  const bool tall = m > n;
  const int side = lay.side;
  const long ldg = lay.ldg;
  const float unit = 1.f / scale, unit_q = 1.f / scale_q;      // powers of two
  const auto slot = [&](int i) { return NsMatrix{square + i * lay.g, ldg, 0}; };
  const NsMatrix none{nullptr, 0, 0};
  const bool carries = ns_carries(batch, m, n, steps);
  int cur = 0, rc = 0;
  for (int done = 0; done < steps;) {
    const int len = ns_segment(carries, steps - done);
    const bool last = done + len == steps;
    const NsMatrix xi{x[cur], lay.ldx, 0}, xo{last ? out : x[cur ^ 1], last ? (long)n : lay.ldx, 0};
    const auto diagonal = [&](int slot_i) { return diag + static_cast<long>(slot_i) * batch * side; };
    NsEpilogue eg{};
    eg.alpha = eg.unit = unit;
    eg.c_diag = diagonal(NS_G);
    eg.len = side;
    eg.scale[0] = scale;
    rc = tall ? ns_product<true, true, NS_GRAM>(xi, xi, slot(NS_G), none, batch, 1, side, side, m, eg, sums, status, stream)
              : ns_product<false, false, NS_GRAM>(xi, xi, slot(NS_G), none, batch, 1, side, side, n, eg, sums, status, stream);
    if (rc) return rc;
    // P of the G at hand; with `q` also a I + P
    const auto poly = [&](bool q) {
      NsEpilogue e{};
      e.e = reinterpret_cast<const __half*>(square + NS_G * lay.g);
      e.e_batch = side * ldg;
      e.lde = e.e_cols = (int)ldg;
      e.alpha = c * unit;
      e.coef = b;
      e.diag = diagonal(NS_P);
      e.e_diag = diagonal(NS_G);
      e.c_diag = diagonal(NS_Q);
      e.len = side;
      e.scale[0] = scale;
      e.a = a;
      e.b = b;
      e.c = c;
      e.unit = unit;
      e.also = q ? scale_q * unit : 0.f;
      return ns_product<false, false, NS_POLY>(slot(NS_G), slot(NS_G), slot(NS_P), q ? slot(NS_Q) : none, batch, 1, side, side, side, e, sums,
                                               status, stream);
    };
    // slot `to` = (a I + P) slot `from`, with a second pair of slots (products of Q) where `from2` says so
    const auto carry = [&](int from, int to, int from2, int to2) {
      NsEpilogue e{};
      const int pairs = from2 ? 2 : 1;
      NsMatrix y = slot(from), z = slot(to);
      y.pair_bytes = (from2 - from) * lay.g;
      z.pair_bytes = (to2 - to) * lay.g;
      e.e = static_cast<const __half*>(y.p);
      e.e_batch = side * ldg;
      e.e_pair = y.pair_bytes / 2;
      e.lde = e.e_cols = (int)ldg;
      e.alpha = unit;
      e.coef = a;
      e.diag = diagonal(NS_P);
      e.e_diag = diagonal(from);
      e.c_diag = diagonal(to);
      e.e_diag_pair = static_cast<long>(from2 - from) * batch * side;
      e.c_diag_pair = static_cast<long>(to2 - to) * batch * side;
      e.len = side;
      e.scale[0] = from >= NS_Q ? scale_q : scale;
      e.scale[1] = scale_q;
      e.unit = unit;
      return ns_product<false, false, NS_CARRY>(slot(NS_P), y, z, none, batch, pairs, side, side, side, e, sums, status, stream);
    };
    NsEpilogue eu{};
    eu.len = side;
    eu.e = static_cast<const __half*>(xi.p);
    eu.e_batch = m * lay.ldx;
    eu.lde = eu.e_cols = (int)lay.ldx;
    eu.unit = unit;
    eu.out = static_cast<__nv_bfloat16*>(out);
    eu.last = last;
    if (last) {
      eu.master = apply.master;
      eu.p = apply.p;
      eu.keep = apply.keep;
      eu.step = apply.step;
    }
    int q = NS_P;                              // the matrix that X is multiplied by
    if (len == 1) {
      if ((rc = poly(false))) return rc;
      eu.alpha = unit;
      eu.coef = a;
    } else {
      q = NS_Q;
      int spare = NS_Q + 1;
      if ((rc = poly(true)) || (rc = carry(NS_G, NS_T, 0, 0)) || (rc = carry(NS_T, NS_G, 0, 0))) return rc;
      for (int k = 1; k < len; ++k) {
        if ((rc = poly(false))) return rc;
        rc = k < len - 1 ? carry(NS_G, NS_T, q, spare) : carry(q, spare, 0, 0);
        if (rc || (k < len - 1 && (rc = carry(NS_T, NS_G, 0, 0)))) return rc;
        const int t = q;
        q = spare;
        spare = t;
      }
      eu.alpha = unit_q;
      eu.coef = 0.f;
      eu.rounded = scale_q;
    }
    eu.diag = diagonal(q);
    rc = tall ? ns_product<false, false, NS_UPDATE_T>(xi, slot(q), xo, none, batch, 1, m, n, side, eu, sums, status, stream)
              : ns_product<false, true, NS_UPDATE>(slot(q), xi, xo, none, batch, 1, m, n, side, eu, sums, status, stream);
    if (rc) return rc;
    done += len;
    cur ^= 1;
  }
  return 0;
}

static bool ns_sizes_ok(long batch, long m, long n) {
  return batch >= 1 && m >= 1 && n >= 1 && batch < 1L << 16 && m < 1L << 24 && n < 1L << 24;
}

}  // namespace kb

// Bytes of workspace (256-byte aligned) of the calls below, negative for sizes that they refuse.
extern "C" long kb_newton_schulz_bytes(long batch, long m, long n) {
  return kb::ns_sizes_ok(batch, m, n) ? kb::NsLayout((int)batch, (int)m, (int)n).total : -1;
}
// Kernels that a call of the functions below launches for a batch (the optimizer step: one more unless kb_muon_fuses).
extern "C" int kb_newton_schulz_launches(int batch, int m, int n, int steps) {
  const int side = m < n ? m : n;
  const int gram = kb::ns_plan(kb::NS_GRAM, batch, side, side, m < n ? n : m).parts > 1 ? 2 : 1;
  const bool carries = kb::ns_carries(batch, m, n, steps);
  int launches = 2;
  for (int done = 0; done < steps;) {
    const int len = kb::ns_segment(carries, steps - done);
    launches += gram + (len == 1 ? 2 : 3 * len);
    done += len;
  }
  return launches;
}
// out [batch, m, n] (bf16, 16-byte aligned) = x (fp32 or bf16, contiguous) after `steps` Newton-Schulz steps.  scale: a power of
// two under which every entry of the iterates, of G and of P fits into fp16; scale_q: one for the products of up to three a I + P.
extern "C" int kb_newton_schulz(const void* x, int bf16, int batch, int m, int n, float a, float b, float c, int steps, float eps,
                                float scale, float scale_q, void* out, void* work, int* status, cudaStream_t stream) {
  if (!kb::ns_sizes_ok(batch, m, n) || steps < 1 || !x || !out || !work || reinterpret_cast<uintptr_t>(out) % 16 ||
      reinterpret_cast<uintptr_t>(work) % 256)
    return 7;
  const kb::NsSource src{x, nullptr, nullptr, 0.f, bf16 != 0, false};
  return kb::newton_schulz(src, kb::MuonApply{}, batch, m, n, a, b, c, steps, eps, scale, scale_q, out, static_cast<uint8_t*>(work),
                           status, stream);
}
// Whether the last product of the optimizer step also updates the weights (no kernel of their own): rows of whole 16-byte units.
extern "C" int kb_muon_fuses(const void* master, const void* p, int n) {
  return n % 8 == 0 && reinterpret_cast<uintptr_t>(master) % 16 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}
// One optimizer step of a [m, n] matrix: mom <- beta mom + gs g;  o = Newton-Schulz of (nesterov: gs g + beta mom) or mom;
// master <- keep * master - step * o;  p = bf16(master).  gs: *grad_scale, 1 where that is null.
extern "C" int kb_muon_step(const float* g, float* mom, float* master, void* p, void* o, int m, int n, float beta, int nesterov,
                            float keep, float step, const float* grad_scale, float a, float b, float c, int steps, float eps, float scale,
                            float scale_q, void* work, int* status, cudaStream_t stream) {
  if (!kb::ns_sizes_ok(1, m, n) || steps < 1 || !g || !mom || !master || !p || !o || !work || reinterpret_cast<uintptr_t>(o) % 16 ||
      reinterpret_cast<uintptr_t>(work) % 256)
    return 7;
  const kb::NsSource src{g, mom, grad_scale, beta, false, nesterov != 0};
  const bool fused = kb_muon_fuses(master, p, n);
  kb::MuonApply apply{};
  if (fused) apply = kb::MuonApply{master, static_cast<__nv_bfloat16*>(p), keep, step};
  const int rc = kb::newton_schulz(src, apply, 1, m, n, a, b, c, steps, eps, scale, scale_q, o, static_cast<uint8_t*>(work), status,
                                   stream);
  if (rc || fused) return rc;
  const long count = (long)m * n;
  long blocks = (count + 1023) / 1024;
  blocks = blocks > 148 * 8 ? 148 * 8 : blocks;
  KB_LAUNCH_PDL(kb::muon_apply_kernel, (unsigned)blocks, 256, 0, stream, master, static_cast<__nv_bfloat16*>(p),
                static_cast<const __nv_bfloat16*>(o), count, keep, step);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 2000 + static_cast<int>(e);
}
