// Embedding lookup with a scale, and the gradient of the table by sorted tokens.
//
//   out[t] = s W[id_t]          G[id] += s * sum of dout[t] over the t with id_t = id
//
// The gradient with atomic additions (elementwise.cu) adds the rows of a token as they come, so its bits change from run to run,
// and tokens that make up much of a batch (padding, a frequent word) queue up for the same addresses.  Here the tokens are sorted
// first and each row of the table gets one addition of a sum that was formed in registers:
//
//   1. Stable radix sort of (id, t) by one cluster of eight blocks.  Items stay in the blocks' shared memory; a pass ranks the items
//      of a warp by ballots over the digit's bits, adds up the counts of warps, blocks and digits, and writes every item to its
//      place in the shared memory of the block that owns it.  Tokens of other shards are left out.  Small batches: by counting.
//   2. Blocks take windows of `window` sorted positions and 1024 columns, sum the rows of each token in order and add the sum to the
//      table.  A token whose positions cross the border of a window leaves partial sums: the part that began before the window and
//      the part that goes on after it.
//   3. Such tokens are put together from their partial sums, in order.
//
// Up to 1024 tokens take one kernel for all of it, further below.
//
// The order of additions depends on the tokens alone, so the same inputs give the same bits.  Sums are fp32: of consecutive rows of
// a token, which are put together from front to back.  Batches beyond 65536 tokens are taken in chunks, each of which adds to the table.
//
// What bounds it: memory for the lookup and the sums, latency for the sort and the join.  One B200, us: 8192 x 4096 into 128256 rows
// lookup 18, sort 12, sums 39, join 8; 32768 x 2048, a third of it one token, 21, 14, 24, 12 (the atomic form queues for that row).
#include <cuda_bf16.h>
#include "sm100.cuh"
#include "launch.h"
#include "native_ops.h"
#include "pdl.cuh"
#include "host_utils.h"

namespace kb {

// ----------------------------------------------------------------------------- lookup
// Four tokens a block: their rows are on their way together, since what one row waits for is the latency of its id and of itself.
constexpr int EL_TOKENS = 4;

template <bool VEC>
__global__ void __launch_bounds__(128)
embedding_fwd_kernel(const long* __restrict__ tokens, const __nv_bfloat16* __restrict__ w, __nv_bfloat16* __restrict__ out, long ntok,
                     int H, long first, long rows, float scale) {
  pdl_begin();
  const long t0 = static_cast<long>(blockIdx.x) * EL_TOKENS;
  long id[EL_TOKENS];
#pragma unroll
  for (int k = 0; k < EL_TOKENS; ++k) {
    id[k] = t0 + k < ntok ? tokens[t0 + k] - first : -1;
    if (id[k] >= rows) id[k] = -1;
  }
  if constexpr (VEC) {
    for (int c = threadIdx.x * 8; c < H; c += 128 * 8) {
      uint4 v[EL_TOKENS];
#pragma unroll
      for (int k = 0; k < EL_TOKENS; ++k)
        v[k] = id[k] >= 0 ? __ldg(reinterpret_cast<const uint4*>(w + id[k] * H + c)) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int k = 0; k < EL_TOKENS; ++k) {
        if (scale != 1.f) {
          uint32_t* p = reinterpret_cast<uint32_t*>(&v[k]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            p[j] = id[k] >= 0 ? pack_bf16x2(__uint_as_float(p[j] << 16) * scale, __uint_as_float(p[j] & 0xffff0000u) * scale) : 0u;
        }
        if (t0 + k < ntok) *reinterpret_cast<uint4*>(out + (t0 + k) * H + c) = v[k];
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < EL_TOKENS; ++k) {
      if (t0 + k >= ntok) break;
      for (int c = threadIdx.x; c < H; c += 128)
        out[(t0 + k) * H + c] = __float2bfloat16(id[k] >= 0 ? __bfloat162float(w[id[k] * H + c]) * scale : 0.f);
    }
  }
}

// ----------------------------------------------------------------------------- sort
constexpr int ES_BLOCKS = 8;                   // of a cluster
constexpr int ES_THREADS = 1024;
constexpr int ES_WARPS = ES_THREADS / 32;
constexpr int ES_PER_BLOCK = 8192;             // items
constexpr int ES_MOST = ES_BLOCKS * ES_PER_BLOCK;
constexpr int ES_BITS = 9;                     // of a digit at most: two passes for up to 2^18 rows
constexpr int ES_BINS = 1 << ES_BITS;
constexpr int ES_STEPS = ES_PER_BLOCK / ES_THREADS;        // items a thread at most

__device__ __forceinline__ void st_cluster(uint32_t local, uint32_t rank, uint2 v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster(uint32_t local, uint32_t rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// ids / order [n]: keys below `rows` in ascending order and where they stood; ids behind them are `rows`.  `per`: items of each block
// (a multiple of 32, at most ES_PER_BLOCK, ES_BLOCKS * per >= n); `passes` digits of `bits` (at most ES_BITS) bits hold every key.
// Tokens of other shards leave in the first pass.
__global__ void __cluster_dims__(ES_BLOCKS, 1, 1) __launch_bounds__(ES_THREADS, 1)
embedding_sort_kernel(const long* __restrict__ tokens, int n, int per, long first, long rows, int passes, int bits,
                      uint32_t* __restrict__ ids, uint32_t* __restrict__ order) {
  extern __shared__ uint4 sm[];
  __shared__ uint32_t count[ES_BINS], base[ES_BINS], warp_sum[ES_BINS / 32];
  uint32_t* const hist = reinterpret_cast<uint32_t*>(sm);              // [warps][bins] of 16 bits
  constexpr int HIST_WORDS = ES_BINS / 2;
  uint2 *src = reinterpret_cast<uint2*>(hist + ES_WARPS * HIST_WORDS), *dst = src + per;      // (key, position)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = blockIdx.x;
  const int bins = 1 << bits;
  const int all = n;
  int begin = static_cast<int>(rank) * per, here = max(0, min(per, n - begin));
  pdl_begin();
  for (int i = tid; i < here; i += ES_THREADS) {
    const long id = tokens[begin + i] - first;
    src[i] = make_uint2(static_cast<uint32_t>(id >= 0 && id < rows ? id : rows), begin + i);
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits;
    // a warp takes consecutive items, 32 at a time, so that its ranks follow their order
    const int per_warp = ((per + ES_WARPS - 1) / ES_WARPS + 31) / 32 * 32, steps = per_warp / 32;
    const int used = min(ES_WARPS, (here + per_warp - 1) / per_warp);          // warps with items
    for (int i = tid; i < used * (HIST_WORDS / 4); i += ES_THREADS) sm[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    uint32_t where[ES_STEPS];
    uint16_t* const mine = reinterpret_cast<uint16_t*>(hist + warp * HIST_WORDS);
#pragma unroll
    for (int s = 0; s < ES_STEPS; ++s) {
      const int i = warp * per_warp + s * 32 + lane;
      if (s < steps && warp * per_warp + s * 32 < here) {
        const uint32_t key = i < here ? src[i].x : static_cast<uint32_t>(rows), d = (key >> shift) & (bins - 1);
        const bool in = key < rows;
        uint32_t peers = __ballot_sync(0xffffffffu, in);                       // lanes with the same digit
#pragma unroll
        for (int b = 0; b < ES_BITS; ++b) {
          if (b < bits) {
            const bool one = d >> b & 1u;
            const uint32_t v = __ballot_sync(0xffffffffu, one);
            peers &= one ? v : ~v;
          }
        }
        const uint32_t before = in ? mine[d] : 0u;
        __syncwarp();
        if (in && lane == __ffs(peers) - 1) mine[d] = static_cast<uint16_t>(before + __popc(peers));
        __syncwarp();
        where[s] = before + __popc(peers & ((1u << lane) - 1));
      }
    }
    __syncthreads();
    if (tid < bins / 2 || tid == 0) {                     // counts of the warps before, of the block; two digits a word
      uint32_t sum = 0;
#pragma unroll 4
      for (int w = 0; w < used; ++w) {
        const uint32_t c = hist[w * HIST_WORDS + tid];
        hist[w * HIST_WORDS + tid] = sum;
        sum += c;
      }
      count[2 * tid] = sum & 0xffffu;
      count[2 * tid + 1] = sum >> 16;
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
    if (p == 0) {                                         // what is left, spread evenly again
      n = 0;
#pragma unroll
      for (int w = 0; w < ES_BINS / 32; ++w) n += static_cast<int>(warp_sum[w]);
    }
    const int next_per = max(32, (n + ES_BLOCKS - 1) / ES_BLOCKS);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < ES_STEPS; ++s) {
      const int i = warp * per_warp + s * 32 + lane;
      if (s < steps && i < here) {
        const uint2 item = src[i];
        if (item.x < rows) {
          const uint32_t d = (item.x >> shift) & (bins - 1);
          const uint32_t at = base[d] + mine[d] + where[s], block = at / static_cast<uint32_t>(next_per);
          st_cluster(smem_u32(dst + (at - block * next_per)), block, item);
        }
      }
    }
    cluster_sync_all();
    per = next_per;
    begin = static_cast<int>(rank) * per;
    here = max(0, min(per, n - begin));
    uint2* const t = src;
    src = dst;
    dst = t;
  }
  for (int i = tid; i < here; i += ES_THREADS) {
    ids[begin + i] = src[i].x;
    order[begin + i] = src[i].y;
  }
  for (int i = n + static_cast<int>(rank) * ES_THREADS + tid; i < all; i += ES_BLOCKS * ES_THREADS) ids[i] = static_cast<uint32_t>(rows);
}

// The same for small batches, by counting: the place of a token is the number of smaller ones and of equal ones before it.  A block
// holds all keys, a warp counts for one token, 128 keys at a time.  What a radix pass takes are its many steps; here is one, of n^2
// comparisons, over as many blocks as there are.  One B200, us of the gradient of n x 2048, by a cluster / by counting:
// 1500 18.2 / 14.0, 2048 18.6 / 14.6, 3000 22.0 / 19.0, 4096 24.9 / 23.9.
constexpr int ER_MOST = 4096;                  // tokens
constexpr int ER_THREADS = 256;

__global__ void __launch_bounds__(ER_THREADS)
embedding_rank_kernel(const long* __restrict__ tokens, int n, long first, long rows, uint32_t* __restrict__ ids,
                      uint32_t* __restrict__ order) {
  extern __shared__ uint4 sm[];                // [n rounded up to 128] keys, the largest number behind the last
  uint32_t* const keys = reinterpret_cast<uint32_t*>(sm);
  const int chunks = (n + 127) / 128, lane = threadIdx.x & 31;
  pdl_begin();
#pragma unroll 8
  for (int i = threadIdx.x; i < chunks * 128; i += ER_THREADS) {
    const long id = i < n ? tokens[i] - first : 0;
    keys[i] = i < n ? static_cast<uint32_t>(id >= 0 && id < rows ? id : rows) : 0xffffffffu;
  }
  __syncthreads();
  const int item = blockIdx.x * (ER_THREADS / 32) + (threadIdx.x >> 5);
  if (item >= n) return;
  const uint32_t me = keys[item];
  uint32_t count = 0;
  const auto add = [&](int c, uint32_t below) {
    const uint4 v = sm[c * 32 + lane];
    count += (v.x < below) + (v.y < below) + (v.z < below) + (v.w < below);
  };
  const int own = item / 128;
#pragma unroll 4
  for (int c = 0; c < own; ++c) add(c, me + 1);           // equal keys count too
#pragma unroll 4
  for (int c = own + 1; c < chunks; ++c) add(c, me);
  const uint4 v = sm[own * 32 + lane];
  const uint32_t key[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) count += key[j] < me + (own * 128 + lane * 4 + j < item ? 1u : 0u);
  count = __reduce_add_sync(0xffffffffu, count);
  if (lane == 0) {
    ids[count] = me;
    order[count] = item;
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

// Eight columns of the table's gradient.
template <bool VEC>
__device__ __forceinline__ void load_sums(const float* src, float (&g)[8], int left) {
  if constexpr (VEC) {
    const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
    g[0] = a.x; g[1] = a.y; g[2] = a.z; g[3] = a.w;
    g[4] = b.x; g[5] = b.y; g[6] = b.z; g[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = j < left ? src[j] : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void store_sums(float* dst, const float (&v)[8], int left) {
  if constexpr (VEC) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) dst[j] = v[j];
  }
}

// Eight columns of a row of gradients, and their addition to sums.
template <bool VEC>
__device__ __forceinline__ uint4 load_row(const __nv_bfloat16* src, int left) {
  if constexpr (VEC) return __ldcs(reinterpret_cast<const uint4*>(src));
  uint32_t q[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < left) q[k >> 1] |= static_cast<uint32_t>(__bfloat16_as_ushort(src[k])) << (k & 1 ? 16 : 0);
  return make_uint4(q[0], q[1], q[2], q[3]);
}
__device__ __forceinline__ void add_row(float (&acc)[8], uint4 v) {
  const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    acc[2 * k] += __uint_as_float(q[k] << 16);
    acc[2 * k + 1] += __uint_as_float(q[k] & 0xffff0000u);
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
    // the batch's rows, and the table's rows that its sums go to, are on their way together
    uint4 v[EW_BATCH];
    float old[EW_BATCH][8];
    bool starts = began;
#pragma unroll
    for (int j = 0; j < EW_BATCH; ++j) {
      v[j] = make_uint4(0u, 0u, 0u, 0u);
      const uint32_t me = b + j < len ? id[1 + b + j] : NONE;
      if (me < p.rows) {
        v[j] = load_row<VEC>(p.dout + static_cast<size_t>(pos[b + j]) * p.H + col, left);
        const bool ends = id[2 + b + j] != me;
        if (ends && starts) load_sums<VEC>(p.grad + static_cast<size_t>(me) * p.H + col, old[j], left);
        if (ends) starts = true;
      }
    }
#pragma unroll
    for (int j = 0; j < EW_BATCH; ++j) {
      const uint32_t me = b + j < len ? id[1 + b + j] : NONE;
      if (me < p.rows) {
        add_row(acc, v[j]);
        const bool last = b + j == len - 1, ends = id[2 + b + j] != me;
        if (last || ends) {
          float* dst;
          if (began && ends) {
            dst = p.grad + static_cast<size_t>(me) * p.H + col;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] = fmaf(acc[k], p.scale, old[j][k]);
          } else {
            dst = (began ? p.after : p.before) + static_cast<size_t>(blockIdx.x) * p.H + col;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] *= p.scale;
          }
          store_sums<VEC>(dst, acc, left);
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] = 0.f;
          began = true;
        }
      }
    }
  }
}

// Tokens that cross windows.  A warp looks whether one begins in its window and goes on.  If it ends within the next few windows the
// warp adds up the parts itself; otherwise the block's sixteen warps share them, each a run of consecutive windows, sixteen of them on
// their way at once (eight and eight took 37 us instead of 33 for 8192 x 2048, nine tenths of it one token).  128 columns a block.
constexpr int EC_THREADS = 512;
constexpr int EC_WARPS = EC_THREADS / 32;
constexpr int EC_COLS = 128;
constexpr int EC_SHORT = 8;

// Sum of the parts that windows from .. to - 1 hold of four columns, in order.
template <bool VEC>
__device__ __forceinline__ float4 sum_parts(const EmbeddingSum& p, int from, int to, int col, int left) {
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (left <= 0) return acc;
#pragma unroll 16
  for (int v = from; v < to; ++v) {
    const float* q = p.before + static_cast<size_t>(v) * p.H + col;
    float4 x;
    if constexpr (VEC) x = *reinterpret_cast<const float4*>(q);
    else x = make_float4(q[0], left > 1 ? q[1] : 0.f, left > 2 ? q[2] : 0.f, left > 3 ? q[3] : 0.f);
    acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
  }
  return acc;
}

template <bool VEC>
__global__ void __launch_bounds__(EC_THREADS) embedding_join_kernel(const EmbeddingSum p) {
  __shared__ __align__(16) float part[EC_WARPS][EC_COLS];
  __shared__ int last_of[EC_WARPS];             // last window of a long token that begins in the warp's window, or 0
  pdl_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, W = p.window;
  const int w = blockIdx.x * EC_WARPS + warp, border = (w + 1) * W;     // first position of the next window
  const int col = blockIdx.y * EC_COLS + lane * 4, left = p.H - col;    // four columns
  const uint32_t NONE = 0xffffffffu;
  uint32_t me = NONE;
  bool begins = false;
  if (border < p.n) {
    me = p.ids[border];
    const uint32_t end_here = p.ids[border - 1], first_here = p.ids[border - W], before = w > 0 ? p.ids[border - W - 1] : NONE;
    begins = me < p.rows && end_here == me && !(first_here == me && before == me);
  }
  int last = 0;                                 // windows w + 1 .. last hold `before` parts of the token
  if (begins) {
    // the first window that it does not leave: keys are sorted, so that is where the next border's key differs
    for (int v = w + 1; !last; v += 128) {
      bool stop[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int next = (v + k * 32 + lane + 1) * W;
        stop[k] = next >= p.n || p.ids[next] != me;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t stops = __ballot_sync(0xffffffffu, stop[k]);
        if (!last && stops) last = v + k * 32 + __ffs(stops) - 1;
      }
    }
    if (last - w <= EC_SHORT) {
      float4 sum = sum_parts<VEC>(p, w + 1, last + 1, col, left);
      const float* a = p.after + static_cast<size_t>(w) * p.H + col;
      float* g = p.grad + static_cast<size_t>(me) * p.H + col;
      if constexpr (VEC) {
        if (left > 0) {
          const float4 x = *reinterpret_cast<const float4*>(a), y = *reinterpret_cast<const float4*>(g);
          *reinterpret_cast<float4*>(g) = make_float4(y.x + (x.x + sum.x), y.y + (x.y + sum.y), y.z + (x.z + sum.z), y.w + (x.w + sum.w));
        }
      } else {
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < left) g[k] += a[k] + v[k];
      }
      last = 0;
    }
  }
  if (lane == 0) last_of[warp] = last;
  if (!__syncthreads_or(last)) return;
  for (int i = 0; i < EC_WARPS; ++i) {
    const int end = last_of[i];
    if (!end) continue;                         // the same for the whole block
    const int start = blockIdx.x * EC_WARPS + i, share = (end - start + EC_WARPS - 1) / EC_WARPS;
    const int from = start + 1 + warp * share, to = min(from + share, end + 1);
    *reinterpret_cast<float4*>(&part[warp][lane * 4]) = sum_parts<VEC>(p, from, to, col, left);
    __syncthreads();
    const int c = blockIdx.y * EC_COLS + threadIdx.x;
    if (threadIdx.x < EC_COLS && c < p.H) {
      float sum = p.after[static_cast<size_t>(start) * p.H + c];
#pragma unroll
      for (int k = 0; k < EC_WARPS; ++k) sum += part[k][threadIdx.x];
      p.grad[static_cast<size_t>(p.ids[(start + 1) * W]) * p.H + c] += sum;
    }
    __syncthreads();
  }
}

// ----------------------------------------------------------------------------- few tokens
// The whole gradient of a small batch in one launch.  A block for each token lists the positions that hold it.  Up to EW_BATCH of them
// are summed by the block of the first, groups of threads with columns of their own.  A longer run is spread over the blocks of its
// tokens by columns, and in a block over groups of threads by rows, whose sums are added in order.
//
// What bounds it: latency, of the tokens and then of a few rows.  One B200, us of the gradient of n x 2048, sorted by counting / so: 64
// tokens 5.2 / 2.5, 512 10.4 / 4.4, nine tenths of them one token 9.9 / 5.3, 1024 12.2 / 7.9; 2048 14.6 / 15.5, since every block goes
// through all tokens.
constexpr int EF_MOST = 1024;                  // tokens
constexpr int EF_THREADS = 256;
constexpr int EF_COLS = 512;                   // of a group, short runs
constexpr int EF_LONG_COLS = 128;              // of a block, long runs
constexpr int EF_GROUPS = EF_THREADS / (EF_COLS / 8), EF_LONG_GROUPS = EF_THREADS / (EF_LONG_COLS / 8);

template <bool VEC>
__global__ void __launch_bounds__(EF_THREADS)
embedding_few_kernel(const long* __restrict__ tokens, const __nv_bfloat16* __restrict__ dout, float* __restrict__ grad, int n, int H,
                     long first, long rows, float scale) {
  constexpr int TURNS = EF_MOST / EF_THREADS, WARPS = EF_THREADS / 32;
  __shared__ uint16_t at[EF_MOST];             // the token's positions
  static_assert(TURNS * WARPS == 32, "a count a lane");
  __shared__ int found[32];                    // in each 32 positions
  __shared__ int place;                        // of this block's token among them
  __shared__ __align__(16) float part[EF_LONG_GROUPS - 1][EF_LONG_COLS];
  pdl_begin();
  const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long me = tokens[t] - first;
  if (me < 0 || me >= rows) return;
  uint32_t same[TURNS];                        // lanes of this warp that hold the token
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    const int i = k * EF_THREADS + tid;
    same[k] = k * EF_THREADS < n ? __ballot_sync(0xffffffffu, i < n && tokens[i] - first == me) : 0u;
    if (lane == 0) found[k * WARPS + warp] = __popc(same[k]);
  }
  __syncthreads();
  const int mine = found[lane];
  int before = mine;                           // in the positions before the lane's 32
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, before, i);
    if (lane >= i) before += o;
  }
  const int len = __shfl_sync(0xffffffffu, before, 31);
  before -= mine;
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    if (k * EF_THREADS >= n) break;
    const int p = __shfl_sync(0xffffffffu, before, k * WARPS + warp) + __popc(same[k] & ((1u << lane) - 1)), i = k * EF_THREADS + tid;
    if (same[k] >> lane & 1u) {
      at[p] = static_cast<uint16_t>(i);
      if (i == t) place = p;
    }
  }
  __syncthreads();
  const auto sum = [&](int col, int from, int to, float (&acc)[8]) {
    for (int b = from; b < to; b += EW_BATCH) {
      uint4 v[EW_BATCH];
#pragma unroll
      for (int j = 0; j < EW_BATCH; ++j)
        v[j] = b + j < to ? load_row<VEC>(dout + static_cast<size_t>(at[b + j]) * H + col, H - col) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int j = 0; j < EW_BATCH; ++j)
        if (b + j < to) add_row(acc, v[j]);
    }
  };
  float* const row = grad + me * H;
  const auto finish = [&](int col, float (&acc)[8], const float (&old)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = fmaf(acc[k], scale, old[k]);
    store_sums<VEC>(row + col, acc, H - col);
  };
  if (len <= EW_BATCH) {
    if (place) return;
    const int group = tid / (EF_COLS / 8), c = tid % (EF_COLS / 8) * 8;
    for (int col = (blockIdx.y + gridDim.y * group) * EF_COLS + c; col < H; col += gridDim.y * EF_GROUPS * EF_COLS) {
      float acc[8] = {}, old[8];
      load_sums<VEC>(row + col, old, H - col);
      sum(col, 0, len, acc);
      finish(col, acc, old);
    }
    return;
  }
  const int group = tid / (EF_LONG_COLS / 8), c = tid % (EF_LONG_COLS / 8) * 8;
  const int share = (len + EF_LONG_GROUPS - 1) / EF_LONG_GROUPS, from = group * share, to = min(len, from + share);
  for (int col0 = (place * gridDim.y + blockIdx.y) * EF_LONG_COLS; col0 < H; col0 += len * gridDim.y * EF_LONG_COLS) {
    const int col = col0 + c;
    float acc[8] = {}, old[8];
    if (group == 0 && col < H) load_sums<VEC>(row + col, old, H - col);
    if (col < H) sum(col, from, to, acc);
    if (group > 0) store_sums<true>(&part[group - 1][c], acc, 8);
    __syncthreads();
    if (group == 0 && col < H) {
#pragma unroll
      for (int g = 0; g < EF_LONG_GROUPS - 1; ++g) {
        float more[8];
        load_sums<true>(&part[g][c], more, 8);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] += more[k];
      }
      finish(col, acc, old);
    }
    __syncthreads();                           // the sums have been read
  }
}

// ----------------------------------------------------------------------------- host side
// Sorted positions per block of the sums: 64, fewer where that would be less than 512 windows, whose blocks wait for memory side by
// side.  More windows leave a frequent token in more parts to be joined.  One B200, us, 8192 x 5120: 64 positions 97, 32 86, 16 83,
// 8 85; nine tenths of it one token: 52, 49, 50, 58.  Over 2048 to 65536 tokens, 512 to 5120 columns and none, a third or nine tenths
// of one token, 512 windows take 3 % less than only as many as fill the chip twice (geometric mean), 1024 are as slow as those.
static int sum_window(long n) {
  int w = EW_MOST;
  while (w > EW_BATCH && (n + w - 1) / w < 512) w /= 2;
  return w;
}
static long chunk_bytes(long n, int H) {
  if (n <= EF_MOST) return 0;                  // nothing is kept
  const long windows = (n + sum_window(n) - 1) / sum_window(n);
  return (4L * n + 255) / 256 * 256 * 2 + 2L * windows * H * 4;
}

}  // namespace kb

extern "C" int kb_embedding_fwd(const long* tokens, const void* w, void* out, long ntok, int H, long first, long rows, float scale,
                                cudaStream_t stream) {
  if (ntok <= 0 || H <= 0 || rows <= 0) return 7;
  const bool vec = H % 8 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const long grid = (ntok + kb::EL_TOKENS - 1) / kb::EL_TOKENS;
  if (grid >= 1L << 31) return 7;
  KB_LAUNCH_PDL((vec ? kb::embedding_fwd_kernel<true> : kb::embedding_fwd_kernel<false>), static_cast<unsigned>(grid), 128, 0, stream,
                tokens, static_cast<const __nv_bfloat16*>(w), static_cast<__nv_bfloat16*>(out), ntok, H, first, rows, scale);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 2000 + static_cast<int>(e);
}

// Bytes of workspace (256-byte aligned) of the call below; 0: it takes none.
extern "C" long kb_embedding_sorted_bytes(long ntok, int H) {
  if (ntok <= 0 || H <= 0) return 0;
  const long whole = kb::chunk_bytes(kb::ES_MOST, H), rest = kb::chunk_bytes(ntok % kb::ES_MOST ? ntok % kb::ES_MOST : kb::ES_MOST, H);
  return ntok > kb::ES_MOST && whole > rest ? whole : rest;
}
// Kernels that it launches.
extern "C" int kb_embedding_sorted_launches(long ntok) {
  const long rest = ntok % kb::ES_MOST;
  return static_cast<int>(ntok / kb::ES_MOST * 3 + (rest == 0 ? 0 : rest <= kb::EF_MOST ? 1 : 3));
}
// grad [rows, H] (fp32) += scale * the rows of dout ([ntok, H] bf16) at the tokens' rows; tokens outside first .. first + rows - 1
// are left out.  Batches beyond 65536 tokens are taken in chunks of that many.
extern "C" int kb_embedding_bwd_sorted(const long* tokens, const void* dout, float* grad, long ntok, int H, long first, long rows,
                                       float scale, void* work, cudaStream_t stream) {
  using namespace kb;
  constexpr int MOST = 65535 * EC_COLS;         // columns, one row of blocks for each EC_COLS of them
  if (ntok <= 0 || H <= 0 || H > MOST || rows <= 0 || rows >= 1L << 31 || reinterpret_cast<uintptr_t>(work) % 256 ||
      (!work && ntok > EF_MOST))
    return 7;
  const bool vec = H % 8 == 0 && reinterpret_cast<uintptr_t>(dout) % 16 == 0 && reinterpret_cast<uintptr_t>(grad) % 16 == 0;
  int bits_all = 1;
  while ((rows - 1) >> bits_all) ++bits_all;              // keys 0 .. rows - 1
  const int passes = (bits_all + ES_BITS - 1) / ES_BITS, bits = (bits_all + passes - 1) / passes;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 7;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               ES_WARPS * ES_BINS * 2 + 2 * ES_PER_BLOCK * 8);
    if (e != cudaSuccess) return 1000 + static_cast<int>(e);
    configured[dev] = true;
  }
  for (long at = 0; at < ntok; at += ES_MOST) {
    const int n = static_cast<int>(ntok - at < ES_MOST ? ntok - at : ES_MOST);
    if (n <= EF_MOST) {
      // blocks of a token: two per SM in all (with four, 64 x 8192 takes 3.9 us instead of 3.1, with eight 4.9)
      const int strips = (H + EF_COLS - 1) / EF_COLS, most = 2 * device_sm_count() / n;
      KB_LAUNCH_PDL((vec ? embedding_few_kernel<true> : embedding_few_kernel<false>), dim3(n, strips < most ? strips : most < 1 ? 1 : most),
                    EF_THREADS, 0, stream, tokens + at, static_cast<const __nv_bfloat16*>(dout) + at * H, grad, n, H, first, rows, scale);
      continue;
    }
    const int per = ((n + ES_BLOCKS - 1) / ES_BLOCKS + 31) / 32 * 32;
    const long list = (4L * n + 255) / 256 * 256;
    EmbeddingSum s;
    uint8_t* base = static_cast<uint8_t*>(work);
    uint32_t* ids = reinterpret_cast<uint32_t*>(base);
    uint32_t* order = reinterpret_cast<uint32_t*>(base + list);
    s.window = sum_window(n);
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
    if (n <= ER_MOST) {
      constexpr int ITEMS = ER_THREADS / 32;
      KB_LAUNCH_PDL(embedding_rank_kernel, (n + ITEMS - 1) / ITEMS, ER_THREADS, (n + 127) / 128 * 512, stream, tokens + at, n, first,
                    rows, ids, order);
    } else {
      KB_LAUNCH_PDL(embedding_sort_kernel, ES_BLOCKS, ES_THREADS, ES_WARPS * ES_BINS * 2 + 2 * per * 8, stream, tokens + at, n, per, first,
                    rows, passes, bits, ids, order);
    }
    KB_LAUNCH_PDL((vec ? embedding_window_kernel<true> : embedding_window_kernel<false>), dim3(windows, (H + EW_COLS - 1) / EW_COLS),
                  EW_THREADS, 0, stream, s);
    KB_LAUNCH_PDL((vec ? embedding_join_kernel<true> : embedding_join_kernel<false>),
                  dim3((windows + EC_WARPS - 1) / EC_WARPS, (H + EC_COLS - 1) / EC_COLS), EC_THREADS, 0, stream, s);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 2000 + static_cast<int>(e);
}
