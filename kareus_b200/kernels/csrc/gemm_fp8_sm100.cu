// C = A * B^T of 8-bit matrices with power-of-two scales (fp8_quantize.cu) on pairs of SMs.
//
// The scales are applied by the tensor cores: tcgen05 kind::mxf8f6f4 multiplies each product of 32 elements along K by two
// exponents that lie in tensor memory, one byte for a row of A and one for a row of B.  Blocks of 128 are four such steps with the
// same byte, and a 32-bit column of tensor memory holds the bytes of four blocks, so scales are copied there once per 512 of K and
// the step's descriptor says which byte counts.  The accumulator is fp32 and never leaves tensor memory before the end; with
// scales of any fp32 value it would have to be read, scaled and added in registers for each block.
//
// One 256 x BN tile per two-CTA cluster (cta_group::2), as in gemm_pair_sm100.cu:
//   warp 0      TMA producer of this CTA's halves of A and B and of the scales (its 128 rows of A, all BN rows of B)
//   warp 1      MMA issuer (leader CTA only): scales into tensor memory, then the products; allocates TMEM in both CTAs
//   warps 2..9  epilogue: TMEM → registers → 4 KB of swizzled shared memory per warp → TMA store or (C +=) TMA reduce-add
//
// Tensor memory: two accumulators of 256 columns and the scales do not fit into 512.  The second accumulator starts at column
// 224, so that at BN = 256 the two share 32 columns: the epilogue reads those first, and the main loop of the next tile starts as
// soon as they are read.
//
// What bounds it: at 256 columns the tensor pipe (93 to 96 % of its cycles in long sums) and with it the power limit, 1.35 GHz; 32 KB
// reach an SM per 512 clocks, the 64 bytes a clock that it can take, so narrower tiles wait for loads.  Short sums lose a tenth at
// tile borders, between the last product of a tile and the first of the next.  One B200: 8192 x 28672 x 4096 632 us (3.04 PFLOP/s),
// 8192 x 4096 x 28672 623, fp32 += 28672 x 4096 x 8192 674; 17 x 6144 x 4096 11; 328 x 776 x 1032 7, launch and first loads.
#include "sm100.cuh"
#include "launch.h"
#include "native_ops.h"
#include "pdl.cuh"
#include "host_utils.h"

namespace kb {

constexpr int G8_BM = 256;                     // rows of a tile (128 per CTA)
constexpr int G8_BK = 128;                     // one block of the scales; 128 bytes
constexpr int G8_MAX_STAGES = 16;
constexpr int G8_EPI_WARPS = 8;                // 4 TMEM lane quarters x 2 sets of column slabs
constexpr int G8_THREADS = (2 + G8_EPI_WARPS) * 32;
constexpr int G8_A_BYTES = 128 * G8_BK;        // 16 KB: this CTA's rows of A, where there are that many
constexpr int G8_SF_BYTES = 2048;              // scales of 512 of K: 512 bytes for A, up to 1024 for B, in the first stage of each 512
constexpr int G8_RING = 5 * (2 * G8_A_BYTES + G8_SF_BYTES);
constexpr int G8_STG_BYTES = G8_EPI_WARPS * 4096;
constexpr int G8_SMEM = G8_RING + G8_STG_BYTES + 512 + 1024;
constexpr int G8_ACC1 = 224;                   // column of the second accumulator
constexpr int G8_SF_COL = 480;                 // scales: two buffers of 16 columns (4 for A, 8 for B)
static_assert(G8_SMEM <= 227 * 1024, "shared memory per CTA");

struct Fp8Work {
  int tiles_m, tiles_n, group_m, nk;
  int groups_k;                                // 512-wide groups of scales along K
  int a_rows;                                  // rows of A that a CTA loads: 128, or all there are in whole groups of 8
  __device__ __forceinline__ void coords(int t, int& tm, int& tn) const {
    // m-tiles are taken in groups of `group_m`; inside a group the m index runs fastest
    const int per_group = group_m * tiles_n;
    const int g = t / per_group, first_m = g * group_m, gsz = min(group_m, tiles_m - first_m), r = t - g * per_group;
    tm = first_m + r % gsz;
    tn = r / gsz;
  }
};

// Instruction descriptor of kind::mxf8f6f4 without the ids of the scale bytes: fp32 accumulator, E8M0 scales, K-major operands.
__host__ __device__ constexpr uint32_t make_idesc_mxf8(int M, int N, int fmt_a, int fmt_b) {
  return (static_cast<uint32_t>(fmt_a) << 7) | (static_cast<uint32_t>(fmt_b) << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
         (1u << 23) | (static_cast<uint32_t>(M >> 7) << 27);
}
// D (+)= (A, scales) * (B, scales) over both CTAs of the pair.
__device__ __forceinline__ void umma_mxf8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t tmem_sa,
                                               uint32_t tmem_sb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(tmem_sa), "r"(tmem_sb), "r"(accumulate)
      : "memory");
}
// 512 bytes of shared memory (32 rows of 16) to four columns of tensor memory, in each of the four lane quarters of both CTAs.
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint32_t saddr) {
  uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(128 >> 4) << 32;  // 8-row groups are 128 bytes apart; no swizzle
  d |= static_cast<uint64_t>(1) << 46;
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}

// Tells the leader's MMA thread that this warp has read tensor memory.  Nothing else is handed over, and the order of accesses to
// tensor memory is kept by the tcgen05 fences around the barrier: a release of the cluster's memory, which takes half a microsecond,
// is not needed.
__device__ __forceinline__ void mbar_arrive_tmem(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// NARROW: a bf16 output in tiles of 64 columns, whose epilogue takes slabs of 32 so that both sets of warps have one.
template <bool OUT_F32, bool ACCUM, bool NARROW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(G8_THREADS, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                const __grid_constant__ CUtensorMap tmC, const Fp8Work w, const int M, const int N, const int bn,
                const int whole,
                const uint32_t idesc, void* const C, const long ldc, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + G8_RING + G8_STG_BYTES);   // used in the leader
  uint64_t* empty = full + G8_MAX_STAGES;
  uint64_t* tfull = empty + G8_MAX_STAGES;  // [2]
  uint64_t* tempty = tfull + 2;             // [2] used in the leader
  uint64_t* tshare = tempty + 2;            // shared columns are read; used in the leader
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tshare + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  const int tiles = w.tiles_m * w.tiles_n;
  const int half_n = bn >> 1;
  const int a_bytes = w.a_rows * G8_BK, b_bytes = half_n * G8_BK, stage_bytes = a_bytes + b_bytes;
  // An A of few rows: the MMA reads 128 all the same, of each CTA.  What it finds behind the loaded ones only reaches rows of the
  // accumulator that nobody stores, and lies in this block's shared memory (the stages are followed by 32 KB of staging).
  const bool load_a = rank == 0 || M > 128;
  const int stages = min(G8_MAX_STAGES, G8_RING / (stage_bytes + G8_SF_BYTES));
  uint8_t* const sf = smem + stages * stage_bytes;          // a slot per stage
  const bool shared_cols = bn > G8_ACC1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < G8_MAX_STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2 * G8_EPI_WARPS);
    }
    mbar_init(tshare, 8);
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
    prefetch_tmap(&tmSA);
    prefetch_tmap(&tmSB);
  }
  pdl_begin();

  if (warp == 0) {
    // ------------------------------------------------------------------ producer (each CTA: its own halves)
    if (elect_one()) {
      const uint32_t full0 = cluster_addr(full, 0);
      const uint32_t tx = 2u * b_bytes + (M > 128 ? 2u : 1u) * a_bytes;      // bytes of both CTAs, counted on the leader's barrier
      int s = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        int tm, tn;
        w.coords(t, tm, tn);
        const int m0 = tm * G8_BM + rank * 128, n0 = tn * bn;
        const int sb0 = n0 >> 7, sb_count = ((n0 + bn + 127) >> 7) - sb0;      // blocks of 128 rows that the tile's columns touch
        const uint32_t sf_tx = 2u * (1 + sb_count) * 512;
        for (int kb_ = 0; kb_ < w.nk; ++kb_) {
          if (!mbar_wait(&empty[s], ph, abort_flag, status, ST_TIMEOUT_EMPTY)) { ok = false; break; }
          uint8_t* a_dst = smem + s * stage_bytes;
          uint8_t* b_dst = a_dst + a_bytes;
          const uint32_t bar = full0 + s * 8;
          const bool scales = (kb_ & 3) == 0;
          if (rank == 0) mbar_expect_tx(&full[s], tx + (scales ? sf_tx : 0u));
          const int k0 = kb_ * G8_BK;
          if (load_a) tma_load_2d_pair(a_dst, &tmA, bar, k0, m0);
          tma_load_2d_pair(b_dst, &tmB, bar, k0, n0 + rank * half_n);
          if (scales) {
            uint8_t* d = sf + s * G8_SF_BYTES;
            const int g = kb_ >> 2;
            tma_load_2d_pair(d, &tmSA, bar, 0, (tm * 2 + rank) * w.groups_k + g);
            for (int j = 0; j < sb_count; ++j) tma_load_2d_pair(d + 512 + j * 512, &tmSB, bar, 0, (sb0 + j) * w.groups_k + g);
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
      const uint32_t smem0 = smem_u32(smem), sf0 = smem_u32(sf);
      const uint64_t ad0 = make_smem_desc(smem0, 16, 1024), bd0 = make_smem_desc(smem0 + a_bytes, 16, 1024);
      uint32_t tile_i = 0, group_i = 0;
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step, ++tile_i) {
        int tm, tn;
        w.coords(t, tm, tn);
        const int n0 = tn * bn, sb_count = ((n0 + bn + 127) >> 7) - (n0 >> 7);
        const uint32_t sb_shift = (n0 & 127) >> 5;                             // columns before the tile's first row of B
        const uint32_t buf = tile_i & 1u;
        if (!mbar_wait(&tempty[buf], ((tile_i >> 1) & 1u) ^ 1u, abort_flag, status, ST_TIMEOUT_TMEM_EMPTY)) break;
        if (shared_cols && tile_i > 0 && !mbar_wait(tshare, (tile_i - 1) & 1u, abort_flag, status, ST_TIMEOUT_TMEM_EMPTY)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * G8_ACC1;
        uint32_t sa = 0, sb = 0;
        for (int kb_ = 0; kb_ < w.nk; ++kb_) {
          if (!mbar_wait(&full[s], ph, abort_flag, status, ST_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          if ((kb_ & 3) == 0) {
            sa = tmem_base + G8_SF_COL + (group_i & 1u) * 16;
            sb = sa + 4;
            ++group_i;
            const uint32_t src = sf0 + s * G8_SF_BYTES;
            scales_to_tmem(sa, src);
            for (int j = 0; j < sb_count; ++j) scales_to_tmem(sb + 4 * j, src + 512 + 512 * j);
            sb += sb_shift;
          }
          const uint64_t ad = ad0 + static_cast<uint64_t>(s * (stage_bytes >> 4));
          const uint64_t bd = bd0 + static_cast<uint64_t>(s * (stage_bytes >> 4));
          const uint32_t id = idesc | (static_cast<uint32_t>(kb_ & 3) << 29) | (static_cast<uint32_t>(kb_ & 3) << 4);
#pragma unroll
          for (int k = 0; k < G8_BK / 32; ++k) umma_mxf8_pair(d_tmem, ad + k * 2, bd + k * 2, id, sa, sb, (kb_ > 0 || k > 0) ? 1u : 0u);
          umma_commit_pair(&empty[s]);                              // both CTAs may refill the stage
          if (kb_ == w.nk - 1) umma_commit_pair(&tfull[buf]);       // both CTAs' halves are complete
          if (++s == stages) { s = 0; ph ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3;                   // TMEM lane quarter
    const int h = (warp - 2) >> 2;            // this warp takes the column slabs h, h + 2, ...
    uint8_t* stg = smem + G8_RING + (warp - 2) * 4096;
    constexpr int SLAB = OUT_F32 || NARROW ? 32 : 64;          // output columns of a slab, 64 bytes wide if NARROW, else 128
    constexpr int UNITS = NARROW ? 4 : 8, PER_UNIT = OUT_F32 ? 4 : 8;
    const int swizzle = NARROW ? (lane >> 1) & 3 : lane & 7;   // of the 16-byte units of this thread's row, as TMA expects
    const int slabs = bn / SLAB, mine = (slabs - h + 1) >> 1;  // mine >= 1: no tile has fewer than two slabs
    const uint32_t stg_row = smem_u32(stg) + lane * (UNITS * 16);
    // columns that this warp has read may be overwritten, if a tile comes that does
    const auto hand_over = [&](uint64_t* bar, bool awaited) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && awaited) mbar_arrive_tmem(cluster_addr(bar, 0));
      __syncwarp();                                   // TMEM is read by whole warps
    };
    uint32_t tile_i = 0;
    for (int t = first; t < tiles; t += step, ++tile_i) {
      int tm, tn;
      w.coords(t, tm, tn);
      const uint32_t buf = tile_i & 1u;
      const int row0 = tm * G8_BM + rank * 128 + q * 32;
      if (!mbar_wait_warp(&tfull[buf], (tile_i >> 1) & 1u, abort_flag, status, ST_TIMEOUT_TMEM_FULL)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + buf * G8_ACC1 + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
      for (int j = 0; j < mine; ++j) {
        // the slab with the columns that the other accumulator shares comes first: the last one of the first accumulator, the
        // first one of the second
        const int c = h + 2 * (buf == 0 ? mine - 1 - j : j);
        const bool shared = shared_cols && c == (buf == 0 ? slabs - 1 : 0);
        uint32_t o[4 * UNITS];
        __syncwarp();
        if constexpr (NARROW) {
          uint32_t v[32];
          tmem_ld_32x32(taddr + c * 32, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = pack_bf16x2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
        } else if constexpr (OUT_F32) {
          tmem_ld_32x32(taddr + c * 32, o);
          tmem_ld_wait();
          if (shared) hand_over(tshare, t + step < tiles);
        } else {
          uint32_t v0[32], v1[32];
          // the 32 columns that both accumulators share come first
          if (shared && buf == 0) tmem_ld_32x32(taddr + c * 64 + 32, v1);
          else tmem_ld_32x32(taddr + c * 64, v0);
          if (shared) {
            tmem_ld_wait();
            hand_over(tshare, t + step < tiles);
          }
          if (shared && buf == 0) tmem_ld_32x32(taddr + c * 64, v0);
          else tmem_ld_32x32(taddr + c * 64 + 32, v1);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            o[i] = pack_bf16x2(__uint_as_float(v0[2 * i]), __uint_as_float(v0[2 * i + 1]));
            o[16 + i] = pack_bf16x2(__uint_as_float(v1[2 * i]), __uint_as_float(v1[2 * i + 1]));
          }
        }
        if (j == mine - 1) hand_over(&tempty[buf], t + 2 * step < tiles);
        if (lane == 0) tma_store_wait_read<0>();      // the previous slab has left the staging buffer
        __syncwarp();
#pragma unroll
        for (int i = 0; i < UNITS; ++i)
          st_shared_v4(stg_row + ((i ^ swizzle) << 4), o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        const int col = tn * bn + c * SLAB;
        // a TMA store ends on a 16-byte boundary: the columns after the last whole unit, and all of an output whose rows start
        // elsewhere, are stored one by one
        if (col + SLAB > whole && row0 + lane < M) {
          for (int x = max(whole, col); x < min(N, col + SLAB); ++x) {
            const int i = x - col, unit = i / PER_UNIT, sub = i % PER_UNIT;
            const uint8_t* src = stg + lane * (UNITS * 16) + ((unit ^ swizzle) << 4);
            const size_t at = static_cast<size_t>(row0 + lane) * ldc + x;
            if constexpr (!OUT_F32) static_cast<__nv_bfloat16*>(C)[at] = reinterpret_cast<const __nv_bfloat16*>(src)[sub];
            else if constexpr (ACCUM) static_cast<float*>(C)[at] += reinterpret_cast<const float*>(src)[sub];
            else static_cast<float*>(C)[at] = reinterpret_cast<const float*>(src)[sub];
          }
        }
        __syncwarp();
        if (lane == 0 && row0 < M && col < whole) {   // the tensor map clips what crosses the edge
          if constexpr (ACCUM) tma_reduce_add_2d(&tmC, stg, col, row0);
          else tma_store_2d(&tmC, stg, col, row0);
          tma_store_commit();
        }
      }
    }
    if (lane == 0) tma_store_wait_read<0>();          // nothing in flight out of shared memory at exit
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                 // the peer's MMAs and arrivals no longer touch this CTA
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

template <bool OUT_F32, bool ACCUM, bool NARROW>
static int launch_fp8(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmSA, const CUtensorMap& tmSB, void* C,
                      int M, int N, long ldc, const Fp8Work& w, int bn, uint32_t idesc, int pairs, int* status, cudaStream_t stream) {
  CUtensorMap tmC = tmA;                       // without columns that TMA can store there is no map and none is needed
  const bool rows_ok = ldc % (OUT_F32 ? 4 : 8) == 0 && reinterpret_cast<uintptr_t>(C) % 16 == 0;
  const int whole = rows_ok ? N & ~(OUT_F32 ? 3 : 7) : 0;
  if (whole) {
    const uint64_t dims[2] = {(uint64_t)whole, (uint64_t)M};
    const uint64_t str[1] = {(uint64_t)ldc * (OUT_F32 ? 4 : 2)};
    const uint32_t box[2] = {OUT_F32 || NARROW ? 32u : 64u, 32u};
    const int rc = make_tmap(&tmC, C, OUT_F32 ? 4 : 2, 2, dims, str, box, NARROW ? 2 : 3);
    if (rc) return rc;
  }
  auto kern = gemm_fp8_kernel<OUT_F32, ACCUM, NARROW>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 7;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G8_SMEM);
    if (e != cudaSuccess) return 1000 + static_cast<int>(e);
    configured[dev] = true;
  }
  const int tiles = w.tiles_m * w.tiles_n;
  const int grid = 2 * (tiles < pairs ? tiles : pairs);
  KB_LAUNCH_PDL(kern, grid, G8_THREADS, G8_SMEM, stream, tmA, tmB, tmSA, tmSB, tmC, w, M, N, bn, whole, idesc, C, ldc,
                status);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 2000 + static_cast<int>(e);
}

// Rows of A that a CTA loads.
static int fp8_rows_of_a(int M) { return M < 128 ? (M + 7) / 8 * 8 : 128; }
// Width of the tiles: clocks of a step of 128 are the larger of the tensor cores' (2 per column) and of the loads' (64 bytes a
// clock reach an SM: two per row of A, one per column for B), times the tiles that a pair works through.
static int fp8_tile_columns(int M, int N, int K, int pairs) {
  const long tiles_m = ((long)M + G8_BM - 1) / G8_BM;
  const int nk = (K + G8_BK - 1) / G8_BK, a_rows = fp8_rows_of_a(M);
  int bn = 256;
  double best = 0;
  for (int b = 256; b >= 64; b -= 64) {
    const long tiles = tiles_m * (((long)N + b - 1) / b);
    const double cost = (double)((tiles + pairs - 1) / pairs) * (nk * (double)(b > 2 * a_rows ? 2 * b : 2 * a_rows + b) + 1500.0);
    if (b == 256 || cost < best * 0.97) {
      best = cost;
      bn = b;
    }
  }
  return bn;
}

}  // namespace kb

// Width of the tiles that the call below takes on `sms` SMs.
extern "C" int kb_gemm_fp8_columns(int M, int N, int K, int sms) { return kb::fp8_tile_columns(M, N, K, sms / 2); }
// C [M, N] = A [M, K] * B [N, K]^T: bytes of format 0 (e4m3) or 1 (e5m2) with rows of lda / ldb bytes (multiples of 16), scales as
// kb_fp8_quantize lays them out.  C: bf16 or fp32 (out_f32), rows of ldc elements; accumulate (fp32): +=.
extern "C" int kb_gemm_fp8(const void* A, const void* SA, int fmt_a, long lda, const void* B, const void* SB, int fmt_b, long ldb,
                           void* C, long ldc, int M, int N, int K, int out_f32, int accumulate, int* status, cudaStream_t stream) {
  using namespace kb;
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  constexpr int MOST = 0x7fffffff - 511;       // row and column numbers are ints, those of tiles across the edge too
  if (M <= 0 || N <= 0 || K <= 0 || M > MOST || N > MOST || K > MOST || lda < K || ldb < K || lda % 16 || ldb % 16 || ldc < N ||
      !aligned(A) || !aligned(B) || !aligned(SA) || !aligned(SB) || (fmt_a & ~1) || (fmt_b & ~1) ||
      (accumulate && !out_f32))
    return 7;
  const int pairs = device_sm_count() / 2;
  Fp8Work w;
  w.tiles_m = (M + G8_BM - 1) / G8_BM;
  w.nk = (K + G8_BK - 1) / G8_BK;
  w.groups_k = (w.nk + 3) / 4;
  w.a_rows = fp8_rows_of_a(M);
  const int bn = fp8_tile_columns(M, N, K, pairs);
  w.tiles_n = (N + bn - 1) / bn;
  const long panel = (long)G8_BM * K;          // m-tiles per group: about 24 MB of A rows, 8 to 16 tiles
  long gm = (24L << 20) / panel;
  gm = gm < 8 ? 8 : gm > 16 ? 16 : gm;
  w.group_m = gm < w.tiles_m ? (int)gm : w.tiles_m;
  if ((long)w.tiles_m * w.tiles_n >= 1L << 30) return 7;

  CUtensorMap tmA, tmB, tmSA, tmSB;
  int rc;
  {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)M}, str[1] = {(uint64_t)lda};
    const uint32_t box[2] = {(uint32_t)G8_BK, (uint32_t)w.a_rows};
    if ((rc = make_tmap(&tmA, A, 1, 2, dims, str, box, 3))) return rc;
  }
  {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)N}, str[1] = {(uint64_t)ldb};
    const uint32_t box[2] = {(uint32_t)G8_BK, (uint32_t)bn / 2};
    if ((rc = make_tmap(&tmB, B, 1, 2, dims, str, box, 3))) return rc;
  }
  const uint64_t str[1] = {512};
  const uint32_t box[2] = {128u, 1u};          // 128 words: the scales of 128 rows x 512
  const uint64_t da[2] = {128, (uint64_t)((M + 127) / 128) * w.groups_k}, db[2] = {128, (uint64_t)((N + 127) / 128) * w.groups_k};
  if ((rc = make_tmap(&tmSA, SA, 4, 2, da, str, box, 0))) return rc;
  if ((rc = make_tmap(&tmSB, SB, 4, 2, db, str, box, 0))) return rc;
  const uint32_t idesc = make_idesc_mxf8(G8_BM, bn, fmt_a, fmt_b);
  // bn is a multiple of 64: two slabs of columns a tile at least, of 32 in fp32 and in the narrow form, of 64 in the other
  if (!out_f32 && bn == 64)
    return launch_fp8<false, false, true>(tmA, tmB, tmSA, tmSB, C, M, N, ldc, w, bn, idesc, pairs, status, stream);
  if (!out_f32) return launch_fp8<false, false, false>(tmA, tmB, tmSA, tmSB, C, M, N, ldc, w, bn, idesc, pairs, status, stream);
  if (accumulate) return launch_fp8<true, true, false>(tmA, tmB, tmSA, tmSB, C, M, N, ldc, w, bn, idesc, pairs, status, stream);
  return launch_fp8<true, false, false>(tmA, tmB, tmSA, tmSB, C, M, N, ldc, w, bn, idesc, pairs, status, stream);
}
