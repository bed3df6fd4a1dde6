// kv4.cuh -- the 4-bit paged key/value cache shared by its kernels: where a
// tile's parts lie, where a channel's code sits in its row, and the launch
// helper of the entry points.
//
// The cache is [n_blocks][n_kv_heads][block_size / 16] tiles.  A tile holds 16
// tokens of one KV head in one contiguous piece, so that a bulk copy brings
// everything attention needs of them:
//   K codes [16][D/2] | V codes [16][D/2] | K {scale, min} [D/G][16] | V {scale, min} [D/G][16]
// A code c of a group with {scale, min} stands for c * scale + min.
// The order of a row's channels is the one in which mma.m16n8k16 takes them:
//   K: lane quad member c reads the words c*(D/32) .. of its row in one vector
//      load; word j of them holds channels 32j + 8c .. + 7, so the 32 channels
//      of one chunk j (never more than one group) feed the same two MMAs.
//   V: lane group g reads the words g*(D/64) ..; word s of them holds channels
//      64s + 4g .. + 3 in its low half and 64s + 32 + 4g .. + 3 in its high
//      half, so an 8-wide output tile never spans two groups of 32 either.
#pragma once

#include <algorithm>
#include <cstdint>

#include "device_util.cuh"
#include "nimf_internal.h"

namespace nimf {
namespace kv4 {

constexpr int kTile = 16;  // tokens of a tile
constexpr int kMaxSeqs = 1 << 30;  // requests of a call: searches add two indexes in 32 bits

// Sizes of a cache as the kernels take them.
struct Shape {
  int64_t n_blocks = 0;
  int hkv = 0, d = 0, bs = 0, group = 0;
};

__host__ __device__ constexpr int tile_bytes(int d, int ng) { return kTile * d + 2 * kTile * 8 * ng; }
__host__ __device__ constexpr int v_codes_at(int d) { return kTile * d / 2; }
__host__ __device__ constexpr int k_params_at(int d) { return kTile * d; }
__host__ __device__ constexpr int v_params_at(int d, int ng) { return kTile * d + kTile * 8 * ng; }

// Byte and nibble (0: low) of channel ch in a K or V row of D channels.
__host__ __device__ constexpr int k_byte(int ch, int d) {
  return (((ch % 32) / 8) * (d / 32) + ch / 32) * 4 + (ch % 8) / 2;
}
__host__ __device__ constexpr int v_byte(int ch, int d) {
  return (((ch % 32) / 4) * (d / 64) + ch / 64) * 4 + ((ch % 64) / 32) * 2 + (ch % 4) / 2;
}

// Checks a descriptor (NIMF_ERR_SHAPE / NIMF_ERR_ARG) and copies it.
int check_desc(const nimf_kv4_desc* desc, const char* who, Shape* out);

int stream_of(void* stream, cudaStream_t* st);

// Lets a kernel use `bytes` of dynamic shared memory (asked of the driver once
// per kernel and device binding).
int allow_smem(const void* kern, int bytes);

// Launch with programmatic dependent launch allowed; every kernel launched
// this way waits (griddep_wait) before it touches memory.  One does not:
// attn_kernel<.., BESIDE = true>, which only tc_kernel precedes, relies on that
// kernel having waited before it lets dependents start.
template <typename... KArgs, typename... Args>
int launch(void (*kern)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t st,
           unsigned cluster, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  NIMF_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, ((KArgs)args)...));
  return NIMF_OK;
}

// Cluster barrier halves (every thread of every CTA of the cluster).
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// Inclusive sum over the block's threads (blockDim.x a multiple of 32, at most
// 1024) of one value each; *total receives the block's sum.  sh: 33 words.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* sh, T* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = v;
  __syncthreads();
  if (warp == 0) {
    T w = lane < nw ? sh[lane] : (T)0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    sh[lane] = w;
  }
  __syncthreads();
  if (warp > 0) v += sh[warp - 1];
  *total = sh[nw - 1];
  return v;
}

// ------------------------------------------------------------------ attention
// What attention's kernels are given.
struct Args {
  const uint8_t* cache;
  const float* q;
  const int32_t* cu_rows;     // NULL: one row per sequence
  const int32_t* lens;
  const int32_t* table;
  float* out;
  unsigned char* ws;
  int* err;
  int64_t n_seqs, rows, width, n_blocks;
  int h, hkv, r, bs;
  float scale2;               // softmax scale * log2(e)
  int uncut, wide;            // no segment is shared by CTAs; 64-bit sums of units
  int big;                    // sequences with more rows a KV head than this go to kv4_tc.cu (INT32_MAX: none)
  int sms;                    // CTAs of kv4_tc.cu that run at once
};

// Sequence b as the kernels see it: its rows [row0, row0 + n) and its cached
// tokens, both held inside the caller's buffers.
struct Seq {
  int64_t row0;
  int n, len;
};
__device__ __forceinline__ Seq seq_of(const Args& a, int64_t b) {
  Seq s;
  int64_t e;
  const int32_t* cu = a.cu_rows;
  asm volatile("" : "+l"(cu));  // opaque: loops are not to be copied for either case
  if (cu) {
    s.row0 = min((int64_t)max(cu[b], 0), a.rows);
    e = min((int64_t)max(cu[b + 1], 0), a.rows);
  } else {
    s.row0 = min(b, a.rows);
    e = min(b + 1, a.rows);
  }
  s.n = (int)max(e - s.row0, (int64_t)0);
  s.len = (int)min((int64_t)max(a.lens[b], 0), a.width * a.bs);
  return s;
}
// a / b for a >= 0, b > 0: the 32-bit division, a quarter of the 64-bit one's
// time, wherever it serves.
__device__ __forceinline__ int64_t quot(int64_t a, int64_t b) {
  return ((uint64_t)(a | b) >> 32) ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
// 2^(e - 127) for an exponent field e clamped to the normal range.
__device__ __forceinline__ float pow2_field(int e) {
  return __int_as_float(max(1, min(254, e)) << 23);
}
__device__ __forceinline__ int exp_field(float x) { return (__float_as_int(x) >> 23) & 255; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
  return d;
}
// Joins partial results of one row (maximum, sum, unnormalised outputs of this
// lane's V channels), in the order in which they are taken.
template <int V>
struct Merged {
  float m = -INFINITY, l = 0.f, o[V] = {};
  __device__ __forceinline__ void take(float pm, float pl, const float (&po)[V]) {
    const float top = fmaxf(m, pm), ref = top == -INFINITY ? 0.f : top;
    const float f = ex2(m - ref), pf = ex2(pm - ref);
    m = top;
    l = fmaf(l, f, pl * pf);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = fmaf(o[i], f, po[i] * pf);
  }
};
template <int V>
__device__ __forceinline__ void load_v(const float* p, float (&x)[V]) {
  if constexpr (V == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    x[0] = v.x;
    x[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 v = reinterpret_cast<const float4*>(p)[i];
      x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
    }
  }
}
template <int V>
__device__ __forceinline__ void store_v(float* p, const float (&x)[V], float f) {
  if constexpr (V == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(x[0] * f, x[1] * f);
  } else {
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      reinterpret_cast<float4*>(p)[i] = make_float4(x[4 * i] * f, x[4 * i + 1] * f, x[4 * i + 2] * f, x[4 * i + 3] * f);
  }
}

// Attention of sequences with more than a.big rows a KV head, on tcgen05
// (kv4_tc.cu): an item is 128 rows of one KV head.  Items run in waves of a CTA
// an SM; those of a last wave that half fills the SMs or less are cut into parts
// of their tokens, as many as run at once.  A part is the rows' outputs, maxima
// and sums.
constexpr int kTcRows = 128;
__device__ __forceinline__ int big_tiles(const Args& a, int n) {
  return n * a.r > a.big ? (n * a.r + kTcRows - 1) / kTcRows : 0;
}
struct Waves {
  int items, whole, cut;        // items; those of full waves; parts of each of the others
  __device__ __forceinline__ Waves(const Args& a, int n) {
    items = n;
    whole = n / a.sms * a.sms;
    cut = a.sms / max(n - whole, 1);
    if (cut < 1 || n == whole) cut = 1;
  }
  // Parts of an item, each of four tiles of tokens or more.
  __device__ __forceinline__ int parts(int item, int token_tiles) const {
    return item < whole ? 1 : max(1, min(cut, token_tiles / 4));
  }
};
__host__ __device__ constexpr size_t tc_part_floats(int d) { return (size_t)kTcRows * (d + 2); }
// The sequence and its tile of rows of index i, counted from the end (the last
// rows see most tokens: the longest go first), and the number of all tiles.
// Every lane of a warp gets them.
__device__ __forceinline__ bool find_tile(const Args& a, int index, int& b, int& tile, int& total) {
  const int lane = threadIdx.x & 31;
  total = 0;
  for (int64_t b0 = 0; b0 < a.n_seqs; b0 += 32) {
    const int64_t x = b0 + lane;
    total += __reduce_add_sync(0xffffffffu, x < a.n_seqs ? big_tiles(a, seq_of(a, x).n) : 0);
  }
  if (index >= total) return false;
  int want = total - 1 - index, base = 0;
  for (int64_t b0 = 0; b0 < a.n_seqs; b0 += 32) {
    const int64_t x = b0 + lane;
    const int t = x < a.n_seqs ? big_tiles(a, seq_of(a, x).n) : 0;
    int upto = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, base + upto > want);
    if (past) {
      const int who = __ffs(past) - 1;
      tile = want - base - __shfl_sync(0xffffffffu, upto - t, who);
      b = (int)b0 + who;
      return true;
    }
    base += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}
// Tokens that some row of the tile sees.
__device__ __forceinline__ int tile_len(const Args& a, const Seq& s, int tile) {
  const int rows = min(kTcRows, s.n * a.r - tile * kTcRows);
  const int last_tok = (int)((uint32_t)(tile * kTcRows + rows - 1) / (uint32_t)a.r);
  return max(0, min(s.len, s.len - s.n + last_tok + 1));
}

// Head dims served, workspace, items that a call may have at most, launch.
bool tc_serves(int d);
size_t tc_ws_bytes(int d);
int64_t tc_items(const Args& a);
int run_tc(const Args& a, int d, int ng, unsigned char* ws, cudaStream_t st);

}  // namespace kv4
}  // namespace nimf
