// Embedding lookup with a scale, and the gradient of the table by sorted tokens.
//
//   out[t] = s W[id_t]          G[id] += s * sum of dout[t] over the t with id_t = id, in order of t
//
// The gradient with atomic additions (elementwise.cu) adds the rows of a token as they come, so its bits change from run to run,
// and tokens that make up much of a batch (padding, a frequent word) queue up for the same addresses.  Here the tokens are sorted
// first and each row of the table gets one addition of a sum that was formed in registers:
//
//   1. Stable radix sort of (id, t) by one cluster of eight blocks.  Keys and positions stay in the blocks' shared memory; a pass
//      ranks the items of a warp by __match_any, adds up the counts of warps, blocks and digits, and writes every item to its place
//      in the shared memory of the block that owns it.  Tokens of other shards get the key `rows` and end up behind the others.
//   2. Blocks take windows of `window` sorted positions and 1024 columns, sum the rows of each token in order and add the sum to the
//      table.  A token whose positions cross the border of a window leaves partial sums: the part that began before the window and
//      the part that goes on after it.
//   3. Such tokens are put together from their partial sums, in order.
//
// The order of additions depends on the tokens alone, so the same inputs give the same bits.  Sums are fp32.
#include <cuda_bf16.h>
#include "sm100.cuh"
#include "launch.h"
#include "native_ops.h"
#include "pdl.cuh"
#include "host_utils.h"

namespace kb {

// ----------------------------------------------------------------------------- lookup
template <bool VEC>
__global__ void __launch_bounds__(128)
embedding_scaled_kernel(const long* __restrict__ tokens, const __nv_bfloat16* __restrict__ w, __nv_bfloat16* __restrict__ out, long ntok,
                        int H, long first, long rows, float scale) {
  pdl_begin();
  for (long t = blockIdx.x; t < ntok; t += gridDim.x) {
    const long id = tokens[t] - first;
    const bool inside = id >= 0 && id < rows;
    const __nv_bfloat16* src = w + (inside ? id : 0) * H;
    __nv_bfloat16* dst = out + t * H;
    if constexpr (VEC) {
      for (int c = threadIdx.x * 8; c < H; c += 128 * 8) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (inside) {
          v = *reinterpret_cast<const uint4*>(src + c);
          uint32_t* p = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = pack_bf16x2(__uint_as_float(p[j] << 16) * scale, __uint_as_float(p[j] & 0xffff0000u) * scale);
        }
        *reinterpret_cast<uint4*>(dst + c) = v;
      }
    } else {
      for (int c = threadIdx.x; c < H; c += 128) dst[c] = __float2bfloat16(inside ? __bfloat162float(src[c]) * scale : 0.f);
    }
  }
}

// ----------------------------------------------------------------------------- sort
constexpr int ES_BLOCKS = 8;                   // of a cluster
constexpr int ES_THREADS = 1024;
constexpr int ES_WARPS = ES_THREADS / 32;
constexpr int ES_PER_BLOCK = 8192;             // items
constexpr int ES_MOST = ES_BLOCKS * ES_PER_BLOCK;
constexpr int ES_BINS = 256;
constexpr int ES_STEPS = ES_PER_BLOCK / ES_THREADS;        // items a thread at most

__device__ __forceinline__ void st_cluster(uint32_t local, uint32_t rank, uint32_t v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster(uint32_t local, uint32_t rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// ids / order [n]: keys in ascending order and where they stood.  `per`: items of a block (a multiple of 32, at most ES_PER_BLOCK,
// ES_BLOCKS * per >= n); `passes` digits of `bits` (at most 8) bits hold every key 0 .. rows.
__global__ void __cluster_dims__(ES_BLOCKS, 1, 1) __launch_bounds__(ES_THREADS, 1)
embedding_sort_kernel(const long* __restrict__ tokens, int n, int per, long first, long rows, int passes, int bits,
                      uint32_t* __restrict__ ids, uint32_t* __restrict__ order) {
  extern __shared__ uint32_t sm[];
  __shared__ uint32_t count[ES_BINS], base[ES_BINS], warp_sum[ES_BINS / 32];
  uint32_t* const hist = sm;                              // [warps][bins]
  uint32_t *src = sm + ES_WARPS * ES_BINS, *dst = src + 2 * per;       // keys, positions
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = blockIdx.x;
  const int begin = static_cast<int>(rank) * per, here = max(0, min(per, n - begin));
  // a warp takes consecutive items, 32 at a time, so that its ranks follow their order
  const int per_warp = ((per + ES_WARPS - 1) / ES_WARPS + 31) / 32 * 32, steps = per_warp / 32;
  const int bins = 1 << bits;
  pdl_begin();
  for (int i = tid; i < here; i += ES_THREADS) {
    const long id = tokens[begin + i] - first;
    src[i] = static_cast<uint32_t>(id >= 0 && id < rows ? id : rows);
    src[per + i] = begin + i;
  }
  cluster_sync_all();
  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits;
    for (int i = tid; i < ES_WARPS * bins; i += ES_THREADS) hist[(i >> bits) * ES_BINS + (i & (bins - 1))] = 0;
    __syncthreads();
    uint32_t where[ES_STEPS];
#pragma unroll
    for (int s = 0; s < ES_STEPS; ++s) {
      if (s < steps) {
        const int i = warp * per_warp + s * 32 + lane;
        const bool in = i < here;
        const uint32_t d = in ? (src[i] >> shift) & (bins - 1) : ES_BINS;
        const uint32_t peers = __match_any_sync(0xffffffffu, d);
        uint32_t* h = hist + warp * ES_BINS + (in ? d : 0);
        const uint32_t before = in ? *h : 0;
        __syncwarp();
        if (in && lane == __ffs(peers) - 1) *h = before + __popc(peers);
        __syncwarp();
        where[s] = before + __popc(peers & ((1u << lane) - 1));
      }
    }
    __syncthreads();
    if (tid < bins) {                                     // counts of the warps before, of the block
      uint32_t sum = 0;
      for (int w = 0; w < ES_WARPS; ++w) {
        const uint32_t c = hist[w * ES_BINS + tid];
        hist[w * ES_BINS + tid] = sum;
        sum += c;
      }
      count[tid] = sum;
    }
    cluster_sync_all();
    uint32_t total = 0, before = 0;                       // of this digit in the cluster, in the blocks before
    if (tid < bins) {
#pragma unroll
      for (int b = 0; b < ES_BLOCKS; ++b) {
        const uint32_t c = ld_cluster(smem_u32(&count[tid]), b);
        if (b < static_cast<int>(rank)) before += c;
        total += c;
      }
    }
    uint32_t scan = total;                                // digits before: within the warp, then across warps
    if (warp < ES_BINS / 32) {
#pragma unroll
      for (int i = 1; i < 32; i <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, scan, i);
        if (lane >= i) scan += o;
      }
      if (lane == 31) warp_sum[warp] = scan;
    }
    __syncthreads();
    if (tid < bins) {
      uint32_t add = 0;
      for (int w = 0; w < warp; ++w) add += warp_sum[w];
      base[tid] = add + scan - total + before;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < ES_STEPS; ++s) {
      const int i = warp * per_warp + s * 32 + lane;
      if (s < steps && i < here) {
        const uint32_t key = src[i], d = (key >> shift) & (bins - 1);
        const uint32_t at = base[d] + hist[warp * ES_BINS + d] + where[s];
        const uint32_t block = at / static_cast<uint32_t>(per), slot = at - block * per;
        const uint32_t to = smem_u32(dst + slot);
        st_cluster(to, block, key);
        st_cluster(to + per * 4, block, src[per + i]);
      }
    }
    cluster_sync_all();
    uint32_t* const t = src;
    src = dst;
    dst = t;
  }
  for (int i = tid; i < here; i += ES_THREADS) {
    ids[begin + i] = src[i];
    order[begin + i] = src[per + i];
  }
}

// ----------------------------------------------------------------------------- sums
constexpr int EW_THREADS = 128;
constexpr int EW_COLS = EW_THREADS * 8;
constexpr int EW_MOST = 64;                    // largest window
constexpr int EW_BATCH = 8;                    // rows on their way at once

struct EmbeddingSum {
  const __nv_bfloat16* dout;   // rows of this chunk's tokens
  const uint32_t *ids, *order;
  float* grad;                 // [rows, H]
  float *before, *after;       // [windows][H]: parts of tokens that began before the window / that go on after it
  int n, H, window;
  uint32_t rows;
  float scale;
};

template <bool VEC>
__device__ __forceinline__ void flush(float* dst, const float (&acc)[8], int left, bool add) {
  if constexpr (VEC) {
    if (add) {
      red_add_f32x4(reinterpret_cast<float4*>(dst), make_float4(acc[0], acc[1], acc[2], acc[3]));
      red_add_f32x4(reinterpret_cast<float4*>(dst) + 1, make_float4(acc[4], acc[5], acc[6], acc[7]));
    } else {
      reinterpret_cast<float4*>(dst)[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) dst[j] = add ? dst[j] + acc[j] : acc[j];
  }
}

template <bool VEC>
__global__ void __launch_bounds__(EW_THREADS) embedding_window_kernel(const EmbeddingSum p) {
  __shared__ uint32_t id[EW_MOST + 2], pos[EW_MOST];      // id[0]: the position before the window
  constexpr uint32_t NONE = 0xffffffffu;
  pdl_begin();
  const int w0 = blockIdx.x * p.window, len = min(p.window, p.n - w0);
  for (int i = threadIdx.x; i < len + 2; i += EW_THREADS) {
    const int at = w0 + i - 1;
    id[i] = at >= 0 && at < p.n ? p.ids[at] : NONE;
  }
  for (int i = threadIdx.x; i < len; i += EW_THREADS) pos[i] = p.order[w0 + i];
  __syncthreads();
  const int col = blockIdx.y * EW_COLS + threadIdx.x * 8, left = p.H - col;
  if (left <= 0) return;
  float acc[8] = {};
  bool began = id[1] != id[0];                            // the token at hand starts in this window
  for (int b = 0; b < len; b += EW_BATCH) {
    if (id[1 + b] >= p.rows) break;                       // tokens of other shards: nothing but those from here on
    uint4 v[EW_BATCH];
#pragma unroll
    for (int j = 0; j < EW_BATCH; ++j) {
      v[j] = make_uint4(0u, 0u, 0u, 0u);
      if (b + j < len && id[1 + b + j] < p.rows) {
        const __nv_bfloat16* src = p.dout + static_cast<size_t>(pos[b + j]) * p.H + col;
        if constexpr (VEC) {
          v[j] = __ldcs(reinterpret_cast<const uint4*>(src));
        } else {
          uint32_t* q = reinterpret_cast<uint32_t*>(&v[j]);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < left) q[k >> 1] |= static_cast<uint32_t>(__bfloat16_as_ushort(src[k])) << (k & 1 ? 16 : 0);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < EW_BATCH; ++j) {
      if (b + j < len && id[1 + b + j] < p.rows) {
        const uint32_t q[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          acc[2 * k] += __uint_as_float(q[k] << 16);
          acc[2 * k + 1] += __uint_as_float(q[k] & 0xffff0000u);
        }
        const uint32_t me = id[1 + b + j];
        const bool last = b + j == len - 1, ends = id[2 + b + j] != me;
        if (last || ends) {
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] *= p.scale;
          if (began && ends) flush<VEC>(p.grad + static_cast<size_t>(me) * p.H + col, acc, left, true);
          else flush<VEC>((began ? p.after : p.before) + static_cast<size_t>(blockIdx.x) * p.H + col, acc, left, false);
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] = 0.f;
          began = true;
        }
      }
    }
  }
}

// Tokens that cross windows: block x looks whether one begins in window x and goes on, and adds up its parts.  Eight warps take
// consecutive runs of the windows behind the first, 128 columns a block.
constexpr int EC_THREADS = 256;
constexpr int EC_COLS = 128;

__global__ void __launch_bounds__(EC_THREADS) embedding_join_kernel(const EmbeddingSum p, int windows) {
  __shared__ float part[EC_THREADS / 32][EC_COLS];
  __shared__ int end;
  pdl_begin();
  const int w = blockIdx.x, W = p.window, border = (w + 1) * W;         // first position of the next window
  if (border >= p.n) return;
  const uint32_t me = p.ids[border];
  if (me >= p.rows || p.ids[border - 1] != me) return;
  if (p.ids[border - W] == me && w > 0 && p.ids[border - W - 1] == me) return;   // it began before this window
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) end = windows;
  __syncthreads();
  // the first window from w + 1 on that the token does not leave: keys are sorted, so that is where the next border's key differs
  for (int v = w + 1; v < windows; v += EC_THREADS) {
    const int mine = v + static_cast<int>(threadIdx.x), next = (mine + 1) * W;
    const bool stops = mine < windows && (next >= p.n || p.ids[next] != me);
    if (stops) atomicMin(&end, mine);
    if (__syncthreads_or(stops)) break;
  }
  const int last = min(end, windows - 1), many = last - w;              // windows w + 1 .. last hold `before` parts
  const int share = (many + EC_THREADS / 32 - 1) / (EC_THREADS / 32);
  const int col = blockIdx.y * EC_COLS + lane;                          // columns col, + 32, + 64, + 96
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int from = w + 1 + warp * share, to = min(from + share, last + 1);
#pragma unroll 4
  for (int v = from; v < to; ++v) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + 32 * k < p.H) acc[k] += p.before[static_cast<size_t>(v) * p.H + col + 32 * k];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) part[warp][lane + 32 * k] = acc[k];
  __syncthreads();
  const int c = blockIdx.y * EC_COLS + threadIdx.x;
  if (threadIdx.x < EC_COLS && c < p.H) {
    float sum = p.after[static_cast<size_t>(w) * p.H + c];
#pragma unroll
    for (int i = 0; i < EC_THREADS / 32; ++i) sum += part[i][threadIdx.x];
    p.grad[static_cast<size_t>(me) * p.H + c] += sum;
  }
}

// ----------------------------------------------------------------------------- host side
// Sorted positions per block of the sums: 64 where that fills the chip twice over, fewer for small batches.
static int sum_window(long n, int H) {
  const long cols = (H + EW_COLS - 1) / EW_COLS;
  int w = EW_MOST;
  while (w > EW_BATCH && (n + w - 1) / w * cols < 2L * device_sm_count()) w /= 2;
  return w;
}
static long chunk_bytes(long n, int H) {
  const long windows = (n + sum_window(n, H) - 1) / sum_window(n, H);
  return (4L * n + 255) / 256 * 256 * 2 + 2L * windows * H * 4;
}

}  // namespace kb

extern "C" int kb_embedding_fwd_scaled(const long* tokens, const void* w, void* out, long ntok, int H, long first, long rows, float scale,
                                       cudaStream_t stream) {
  if (ntok <= 0 || H <= 0 || rows <= 0) return 7;
  const bool vec = H % 8 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const unsigned grid = static_cast<unsigned>(ntok < 148 * 16 ? ntok : 148 * 16);
  KB_LAUNCH_PDL((vec ? kb::embedding_scaled_kernel<true> : kb::embedding_scaled_kernel<false>), grid, 128, 0, stream, tokens,
                static_cast<const __nv_bfloat16*>(w), static_cast<__nv_bfloat16*>(out), ntok, H, first, rows, scale);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 2000 + static_cast<int>(e);
}

// Bytes of workspace (256-byte aligned) of the call below.
extern "C" long kb_embedding_sorted_bytes(long ntok, int H) {
  if (ntok <= 0 || H <= 0) return 0;
  const long whole = kb::chunk_bytes(kb::ES_MOST, H), rest = kb::chunk_bytes(ntok % kb::ES_MOST ? ntok % kb::ES_MOST : kb::ES_MOST, H);
  return ntok > kb::ES_MOST && whole > rest ? whole : rest;
}
// grad [rows, H] (fp32) += scale * the rows of dout ([ntok, H] bf16) at the tokens' rows; tokens outside first .. first + rows - 1
// are left out.  Batches beyond 65536 tokens are taken in chunks of that many.
extern "C" int kb_embedding_bwd_sorted(const long* tokens, const void* dout, float* grad, long ntok, int H, long first, long rows,
                                       float scale, void* work, cudaStream_t stream) {
  using namespace kb;
  if (ntok <= 0 || H <= 0 || rows <= 0 || rows >= 1L << 31 || !work || reinterpret_cast<uintptr_t>(work) % 256) return 7;
  const bool vec = H % 8 == 0 && reinterpret_cast<uintptr_t>(dout) % 16 == 0 && reinterpret_cast<uintptr_t>(grad) % 16 == 0;
  int bits_all = 1;
  while (rows >> bits_all) ++bits_all;                    // keys 0 .. rows
  const int passes = (bits_all + 7) / 8, bits = (bits_all + passes - 1) / passes;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 7;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (ES_WARPS * ES_BINS + 4 * ES_PER_BLOCK) * 4);
    if (e != cudaSuccess) return 1000 + static_cast<int>(e);
    configured[dev] = true;
  }
  for (long at = 0; at < ntok; at += ES_MOST) {
    const int n = static_cast<int>(ntok - at < ES_MOST ? ntok - at : ES_MOST);
    const int per = ((n + ES_BLOCKS - 1) / ES_BLOCKS + 31) / 32 * 32;
    const long list = (4L * n + 255) / 256 * 256;
    EmbeddingSum s;
    uint8_t* base = static_cast<uint8_t*>(work);
    uint32_t* ids = reinterpret_cast<uint32_t*>(base);
    uint32_t* order = reinterpret_cast<uint32_t*>(base + list);
    s.window = sum_window(n, H);
    const int windows = (n + s.window - 1) / s.window;
    s.dout = static_cast<const __nv_bfloat16*>(dout) + at * H;
    s.ids = ids;
    s.order = order;
    s.grad = grad;
    s.before = reinterpret_cast<float*>(base + 2 * list);
    s.after = s.before + static_cast<long>(windows) * H;
    s.n = n;
    s.H = H;
    s.rows = static_cast<uint32_t>(rows);
    s.scale = scale;
    KB_LAUNCH_PDL(embedding_sort_kernel, ES_BLOCKS, ES_THREADS, (ES_WARPS * ES_BINS + 4 * per) * 4, stream, tokens + at, n, per, first, rows,
                  passes, bits, ids, order);
    KB_LAUNCH_PDL((vec ? embedding_window_kernel<true> : embedding_window_kernel<false>), dim3(windows, (H + EW_COLS - 1) / EW_COLS),
                  EW_THREADS, 0, stream, s);
    KB_LAUNCH_PDL(embedding_join_kernel, dim3(windows, (H + EC_COLS - 1) / EC_COLS), EC_THREADS, 0, stream, s, windows);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 2000 + static_cast<int>(e);
}
