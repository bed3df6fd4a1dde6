// kv4_pool.cu -- bookkeeping and contents of the 4-bit paged KV cache: block
// tables, slot maps and positions from the requests' lengths, the return of
// finished requests' blocks, the coding of new keys and values into their
// slots, and reading rows back.
#include <cfloat>

#include "kv4.cuh"

namespace nimf {
namespace kv4 {

int check_desc(const nimf_kv4_desc* desc, const char* who, Shape* out) {
  if (!desc) return set_error(NIMF_ERR_ARG, "%s: NULL descriptor", who);
  const int64_t d = desc->head_dim, g = desc->group, bs = desc->block_size;
  if ((d != 64 && d != 128 && d != 256) || (g != 32 && g != 64 && g != 128) || g > d ||
      bs < kTile || bs > 4096 || bs % kTile || desc->n_kv_heads < 1 || desc->n_kv_heads > 65535 ||
      desc->n_blocks < 1 || desc->n_blocks > INT32_MAX / bs)
    return set_error(NIMF_ERR_SHAPE,
                     "%s: n_blocks %lld n_kv_heads %lld head_dim %lld (64, 128 or 256) block_size "
                     "%lld (a multiple of 16, <= 4096) group %lld (32, 64 or 128, <= head_dim); "
                     "n_blocks * block_size below 2^31",
                     who, (long long)desc->n_blocks, (long long)desc->n_kv_heads, (long long)d,
                     (long long)bs, (long long)g);
  out->n_blocks = desc->n_blocks;
  out->hkv = (int)desc->n_kv_heads;
  out->d = (int)d;
  out->bs = (int)bs;
  out->group = (int)g;
  return NIMF_OK;
}

int stream_of(void* stream, cudaStream_t* st) {
  Context* c;
  NIMF_TRY(require_ctx(&c));
  *st = stream ? (cudaStream_t)stream : c->stream;
  return NIMF_OK;
}

int allow_smem(const void* kern, int bytes) {
  struct Done {
    const void* kern;
    int device, bytes;
  };
  constexpr int kKernels = 64;
  static thread_local Done done[kKernels];   // zero: a free place
  const int device = ctx()->device;
  Done* d = done;
  while (d < done + kKernels - 1 && d->kern && d->kern != kern) ++d;
  if (d->kern == kern && d->device == device && d->bytes >= bytes) return NIMF_OK;
  NIMF_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  *d = {kern, device, bytes};
  return NIMF_OK;
}

namespace {

constexpr int kPoolThreads = 1024;

// Block tables and slot maps of one step.  Over the requests in order:
//   rows(b) = [cu(b), cu(b) + new(b))              prefix sum of the new tokens
//   need(b) = ceil((len + new) / bs) - ceil(len / bs)   where the request fits
//   granted = fits and (need == 0 or its inclusive sum of needs <= n_free)
// The sum never falls, so the granted needs are the first ones, and the i-th
// fresh block of the step is free[n_free - 1 - i].
//
// The cost is latency (dependent loads, two scans, a search for each row's
// request), not bytes.  One CTA scans the requests and writes the tables; up to
// kOwnRows rows it also writes the slots (64 requests with one row each: 5 us
// with launch), more are left to a second kernel on all SMs (256
// prompts of 190,000 rows: 12 us, 30 us where a cluster of 8 CTAs did everything).
constexpr int kOwnRows = 4096;

// x / bs for x < 2^31: bs = 16 d, and 2^36 / d rounded up is exact enough.
struct Blocks {
  uint64_t magic;
  uint32_t bs;
  __device__ __forceinline__ uint32_t of(uint32_t x) const { return (uint32_t)((uint64_t)(x >> 4) * magic >> 36); }
};

// The slots and positions of rows [t0, t0 + 128), a warp; the requests' tables
// and lengths are already the new ones.
__device__ __forceinline__ void write_rows(int64_t t0, int n_seqs, int64_t width, Blocks blocks,
                                           int64_t n_blocks, const int32_t* lens_out,
                                           const int32_t* table, int64_t max_rows,
                                           const int32_t* cu_rows, const int32_t* granted,
                                           int32_t* slots, int32_t* positions) {
  const int lane = threadIdx.x & 31;
  // the last request whose first row is <= t0, the same for the warp's last row,
  // then each lane's between them
  int lo = 0, last = 0;
  const int64_t t_end = min(t0 + 127, max_rows - 1);
  for (int step = 1 << (31 - __clz(n_seqs)); step > 0; step >>= 1) {
    const int a = lo + step, b = last + step;
    const int ca = a < n_seqs ? cu_rows[a] : INT32_MAX, cb = b < n_seqs ? cu_rows[b] : INT32_MAX;
    if (ca <= t0) lo = a;
    if (cb <= t_end) last = b;
  }
  int req[4] = {lo, lo, lo, lo};
  if (last > lo)
    for (int step = 1 << (31 - __clz(last - lo)); step > 0; step >>= 1)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int a = min(req[k] + step, last);
        if (cu_rows[a] <= t0 + lane + 32 * k) req[k] = a;
      }
  const int32_t* entry[4];
  int32_t pos[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t t = t0 + lane + 32 * k;
    const int b = req[k];
    const int32_t end = cu_rows[b + 1];
    const bool ok = t < end && granted[b] != 0;
    pos[k] = ok ? lens_out[b] - (end - (int32_t)t) : 0;
    entry[k] = ok ? table + b * width + blocks.of((uint32_t)pos[k]) : nullptr;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t t = t0 + lane + 32 * k;
    const int32_t blk = entry[k] ? *entry[k] : -1;
    const int32_t in = pos[k] - (int32_t)(blocks.of((uint32_t)pos[k]) * blocks.bs);
    if (t < max_rows) {
      const bool there = blk >= 0 && blk < n_blocks;
      slots[t] = there ? blk * (int32_t)blocks.bs + in : -1;
      positions[t] = there ? pos[k] : 0;
    }
  }
}

__global__ void __launch_bounds__(kPoolThreads)
    reserve_kernel(int n_seqs, int64_t width, Blocks blocks, int64_t n_blocks,
                   const int32_t* __restrict__ n_new, const int32_t* lens, int32_t* lens_out,
                   int32_t* table, const int32_t* __restrict__ free_blocks, const int32_t* n_free_in,
                   int32_t* n_free_out, int64_t max_rows, int32_t* cu_rows, int32_t* slots,
                   int32_t* positions, int32_t* granted, int own_rows) {
  __shared__ int64_t sh[33];
  __shared__ int64_t s_off[kPoolThreads];   // fresh blocks before each request of the chunk
  __shared__ int32_t s_have[kPoolThreads];
  __shared__ unsigned long long s_taken;
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x, threads = blockDim.x;
  const uint32_t bs = blocks.bs;
  const int64_t nf = min((int64_t)max(n_free_in[0], 0), n_blocks);
  if (tid == 0) s_taken = 0;
  int64_t cu_base = 0, need_base = 0;
  for (int b0 = 0; b0 < n_seqs; b0 += threads) {
    const int b = b0 + tid;
    const bool live = b < n_seqs;
    const int64_t len = live ? max(lens[b], 0) : 0;
    const int64_t nw = live ? max(n_new[b], 0) : 0;
    int64_t rows_total, need_total;
    const int64_t cu_end = cu_base + block_scan<int64_t>(nw, sh, &rows_total);
    const bool short_enough = len + nw <= (int64_t)INT32_MAX - bs;
    const uint32_t have = blocks.of((uint32_t)min(len, (int64_t)INT32_MAX - bs) + bs - 1);
    const uint32_t total = short_enough ? blocks.of((uint32_t)(len + nw) + bs - 1) : 0;
    const bool fits = live && short_enough && total <= width && cu_end <= max_rows;
    const int64_t need = fits ? total - have : 0;
    const int64_t upto = need_base + block_scan<int64_t>(need, sh, &need_total);
    const bool ok = fits && (need == 0 || upto <= nf);
    const int64_t taken_before = (int64_t)s_taken;
    __syncthreads();
    s_off[tid] = upto - need;
    s_have[tid] = (int32_t)have;
    if (ok && need > 0) atomicMax(&s_taken, (unsigned long long)upto);
    if (live) {
      lens_out[b] = (int32_t)(ok ? len + nw : len);
      granted[b] = ok ? 1 : 0;
      cu_rows[b] = (int32_t)min(cu_end - nw, (int64_t)INT32_MAX);
      if (b == n_seqs - 1) cu_rows[n_seqs] = (int32_t)min(cu_end, (int64_t)INT32_MAX);
    }
    __syncthreads();
    // the chunk's fresh blocks into the tables
    const int cnt = min(threads, n_seqs - b0);
    const int64_t taken = (int64_t)s_taken;
    for (int64_t i0 = max(taken_before, need_base) + tid; i0 < taken; i0 += 4 * threads) {
      int lo[4] = {}, blk[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) blk[k] = i0 + k * threads < taken ? free_blocks[nf - 1 - i0 - k * threads] : 0;
      for (int step = 1 << (31 - __clz(cnt)); step > 0; step >>= 1)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int a = min(lo[k] + step, cnt - 1);
          if (s_off[a] <= i0 + k * threads) lo[k] = a;
        }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k * threads < taken)
          table[(int64_t)(b0 + lo[k]) * width + s_have[lo[k]] + (i0 + k * threads - s_off[lo[k]])] = blk[k];
    }
    cu_base += rows_total;
    need_base += need_total;
    __syncthreads();
  }
  if (tid == 0) {
    n_free_out[0] = (int32_t)(nf - (int64_t)s_taken);
    if (n_seqs == 0) cu_rows[0] = 0;
  }
  if (own_rows)
    for (int64_t t0 = (tid >> 5) * 128; t0 < max_rows; t0 += (threads >> 5) * 128) {
      if (n_seqs > 0) {
        write_rows(t0, n_seqs, width, blocks, n_blocks, lens_out, table, max_rows, cu_rows, granted, slots, positions);
      } else {
        for (int64_t t = t0 + (tid & 31); t < min(t0 + 128, max_rows); t += 32) {
          slots[t] = -1;
          positions[t] = 0;
        }
      }
    }
}

__global__ void __launch_bounds__(256)
    rows_kernel(int n_seqs, int64_t width, Blocks blocks, int64_t n_blocks, const int32_t* __restrict__ lens_out,
                const int32_t* __restrict__ table, int64_t max_rows, const int32_t* __restrict__ cu_rows,
                const int32_t* __restrict__ granted, int32_t* __restrict__ slots, int32_t* __restrict__ positions) {
  griddep_launch_dependents();
  griddep_wait();
  for (int64_t t0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * 128; t0 < max_rows; t0 += (int64_t)gridDim.x * 8 * 128)
    write_rows(t0, n_seqs, width, blocks, n_blocks, lens_out, table, max_rows, cu_rows, granted, slots, positions);
}

// Returns the blocks of the finished requests to the free list, in the order
// of the requests and of their tables, and empties those requests.  One CTA: a
// step finishes few requests.  Latency: table entries are dealt to the threads and
// go straight to their places; a chunk of requests whose tables hold ids that are
// no blocks of the cache is gone through again, in order, without these.  8
// requests of 200 blocks take 3.7 us, 256 of 50 12.6 us (scans in any case 15.4).
__global__ void __launch_bounds__(kPoolThreads)
    release_kernel(int64_t n_seqs, int64_t width, int bs, int64_t n_blocks,
                   const int32_t* __restrict__ finished, int32_t* __restrict__ lens,
                   const int32_t* __restrict__ table, int32_t* __restrict__ free_blocks,
                   int32_t* __restrict__ n_free, int* err) {
  __shared__ int64_t sh[33];
  __shared__ int64_t s_off[kPoolThreads];
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x;
  int64_t top = min((int64_t)max(n_free[0], 0), n_blocks);
  for (int64_t b0 = 0; b0 < n_seqs; b0 += kPoolThreads) {
    const int64_t b = b0 + tid;
    const bool live = b < n_seqs && finished[b] != 0;
    const int64_t pages = live ? min(((int64_t)max(lens[b], 0) + bs - 1) / bs, width) : 0;
    int64_t total;
    const int64_t upto = block_scan<int64_t>(pages, sh, &total);
    s_off[tid] = upto - pages;
    __syncthreads();
    const int cnt = (int)min((int64_t)kPoolThreads, n_seqs - b0);
    auto entry = [&](int64_t i) -> int32_t {    // i of the chunk's table entries in order
      int lo = 0, hi = cnt - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_off[mid] <= i) lo = mid; else hi = mid - 1;
      }
      return table[(b0 + lo) * width + (i - s_off[lo])];
    };
    bool bad = false;
    for (int64_t i = tid; i < total; i += kPoolThreads) {
      const int32_t blk = entry(i);
      bad |= blk < 0 || blk >= n_blocks;
      if (top + i < n_blocks) free_blocks[top + i] = blk;
    }
    if (live) lens[b] = 0;
    int64_t end = top + total;
    if (__syncthreads_or(bad)) {
      if (bad && err) atomicExch(err, 4);
      end = top;
      for (int64_t i0 = 0; i0 < total; i0 += kPoolThreads) {
        const int32_t blk = i0 + tid < total ? entry(i0 + tid) : -1;
        const bool there = blk >= 0 && blk < n_blocks;
        int64_t back;
        const int64_t at = end + block_scan<int64_t>(there, sh, &back) - 1;
        if (there && at < n_blocks) free_blocks[at] = blk;
        end += back;
      }
      __syncthreads();
    }
    if (end > n_blocks && tid == 0 && err) atomicExch(err, 5);  // more blocks returned than there are
    top = min(end, n_blocks);
  }
  if (tid == 0) n_free[0] = (int32_t)top;
}

template <int LANES>
__device__ __forceinline__ float group_min(float v) {
#pragma unroll
  for (int o = LANES >> 1; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int LANES>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = LANES >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// VPL consecutive floats into a row.
template <int VPL>
__device__ __forceinline__ void store_row(float* p, const float (&x)[VPL]) {
  if constexpr (VPL == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
  } else {
#pragma unroll
    for (int i = 0; i < VPL / 4; ++i)
      reinterpret_cast<float4*>(p)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  }
}

// Rotate-half with the row's table entries c and s, each product and sum rounded
// (as nimf_rope_dev).  Lane l holds channels l*VPL ..; the other half of a pair
// is in lane l ^ 16.
template <int VPL>
__device__ __forceinline__ void rotate(float (&x)[VPL], const float (&c)[VPL], const float (&s)[VPL], int lane) {
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const float o = __shfl_xor_sync(0xffffffffu, x[i], 16);
    x[i] = lane >= 16 ? __fadd_rn(__fmul_rn(o, s[i]), __fmul_rn(x[i], c[i]))
                      : __fsub_rn(__fmul_rn(x[i], c[i]), __fmul_rn(o, s[i]));
  }
}

// One group's codes, four bits each, of this lane's VPL channels.
//   scale = (max - min) / 15, code = min(15, round((x - min) / scale)),
// rounded to float at each step, so the codes do not depend on the order of
// anything.  A group with a NaN, an infinity or a range above the largest
// float gets NaN as scale and minimum: all it stands for is NaN.
//
// The quotients are taken as products with 1 / scale, which are off by 2^-18 at
// most here (three roundings of 2^-24, quotients up to 15): where one lies
// within 2^-16 of the middle between two codes, and for scales whose
// reciprocal may overflow, the division decides.
template <int VPL, int LANES>
__device__ __forceinline__ uint32_t code_group(const float (&x)[VPL], int lane, float& scale, float& mn) {
  float mx = x[0];
  mn = x[0];
  bool bad = false;
#pragma unroll
  for (int e = 0; e < VPL; ++e) {
    mn = fminf(mn, x[e]);
    mx = fmaxf(mx, x[e]);
    bad |= !(fabsf(x[e]) <= FLT_MAX);
  }
  mn = __fadd_rn(group_min<LANES>(mn), 0.f);    // -0 and 0 are one minimum, kept as 0
  mx = __fadd_rn(group_max<LANES>(mx), 0.f);
  const unsigned in_group = (LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1u)) << (lane / LANES * LANES);
  bad = (__ballot_sync(0xffffffffu, bad) & in_group) != 0;
  scale = __fdiv_rn(__fsub_rn(mx, mn), 15.0f);
  bad |= !(scale <= FLT_MAX);
  uint32_t code = 0;
  if (!bad && scale > 0.f) {
    bool near = scale < 0x1p-100f;
    const float inv = __frcp_rn(scale);
#pragma unroll
    for (int e = 0; e < VPL; ++e) {
      const float q = __fmul_rn(__fsub_rn(x[e], mn), inv);
      const float r = __fadd_rn(q, 12582912.f);  // its last bits are the nearest integer
      near |= !(fabsf(__fsub_rn(q, __fsub_rn(r, 12582912.f))) < 0.5f - 0x1p-16f);
      code |= (__float_as_uint(r) & 15u) << (4 * e);
    }
    if (near) {
      code = 0;
#pragma unroll 1
      for (int e = 0; e < VPL; ++e) {
        float d = x[0];
#pragma unroll
        for (int i = 1; i < VPL; ++i) d = i == e ? x[i] : d;
        const float r = rintf(__fdiv_rn(__fsub_rn(d, mn), scale));
        code |= (uint32_t)fminf(r, 15.0f) << (4 * e);
      }
    }
  }
  if (bad) scale = mn = __int_as_float(0x7fffffff);
  return code;
}

// A warp takes HB heads of one kind of a row: query heads are rotated, key
// heads rotated and coded, value heads coded.  A lane holds VPL = D/32
// neighbouring channels, a group lies within LANES = G / VPL lanes.
//
// Long batches are bounded by HBM (the queries alone are read and written in
// float32) with HB = 4: four loads go out together, and slot, position and table
// entries are loaded once for them: 8,100 rows of 32 + 8 heads of 128 in groups of
// 32 take 60 us (5.2 TB/s); with their read-back 77 us, 147 with HB = 1.  With
// fewer heads than warps HB = 1 has the shorter way: one row of 32 + 32 heads takes
// 3.8 us with its read-back, 5.0 with HB = 4 (64 rows 6.6 and 6.4).
template <int VPL, int LANES, int HB>
__global__ void __launch_bounds__(256)
    append_kernel(const float* q, float* q_out, int h, const float* __restrict__ k,
                  const float* __restrict__ v, int64_t rows, const int32_t* __restrict__ slots,
                  const int32_t* __restrict__ positions, const float* __restrict__ cos_t,
                  const float* __restrict__ sin_t, int64_t max_seq, uint8_t* __restrict__ cache,
                  int hkv, int bs, int64_t n_slots, int* err) {
  constexpr int D = VPL * 32, NG = 32 / LANES, TB = tile_bytes(D, NG);
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int nq = (h + HB - 1) / HB, nk = (hkv + HB - 1) / HB, per = nq + 2 * nk;
  const int64_t items = rows * per;
  for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items;
       it += (int64_t)gridDim.x * 8) {
    const int64_t t = quot(it, per);
    const int w = (int)(it - t * per);
    const bool is_q = w < nq, is_k = !is_q && w < nq + nk;
    const int h0 = (is_q ? w : is_k ? w - nq : w - nq - nk) * HB, heads = is_q ? h : hkv;
    const float* src = (is_q ? q : is_k ? k : v) + (t * heads + h0) * D + lane * VPL;
    float x[HB][VPL];
#pragma unroll
    for (int i = 0; i < HB; ++i)
      if (HB == 1 || h0 + i < heads) load_v<VPL>(src + i * D, x[i]);
    bool turn = true;
    if (cos_t) {
      const int64_t pos = positions[t];
      turn = pos >= 0 && pos < max_seq;           // otherwise nothing of the row is done
      if (!turn && lane == 0 && err) atomicExch(err, 4);
      if (turn && (is_q || is_k)) {
        float c[VPL], s[VPL];
        load_v<VPL>(cos_t + pos * (D / 2) + (lane & 15) * VPL, c);
        load_v<VPL>(sin_t + pos * (D / 2) + (lane & 15) * VPL, s);
#pragma unroll
        for (int i = 0; i < HB; ++i) rotate<VPL>(x[i], c, s, lane);
      }
    }
    if (is_q) {
      if (turn)
#pragma unroll
        for (int i = 0; i < HB; ++i)
          if (HB == 1 || h0 + i < heads) store_row<VPL>(q_out + (t * h + h0 + i) * D + lane * VPL, x[i]);
      continue;
    }
    const int64_t slot = slots[t];
    if (slot >= n_slots && lane == 0 && err) atomicExch(err, 4);
    if (!turn || slot < 0 || slot >= n_slots) continue;
    const uint32_t blk = (uint32_t)slot / (uint32_t)bs, in_blk = (uint32_t)slot - blk * (uint32_t)bs;
    const int row = in_blk % kTile, tiles = bs / kTile;
    uint8_t* tile = cache + (((int64_t)blk * hkv + h0) * tiles + in_blk / kTile) * TB;
#pragma unroll
    for (int i = 0; i < HB; ++i, tile += (int64_t)tiles * TB) {
      if (HB > 1 && h0 + i >= heads) break;
      float scale, mn;
      const uint32_t code = code_group<VPL, LANES>(x[i], lane, scale, mn);
      uint8_t* codes = tile + (is_k ? 0 : v_codes_at(D)) + row * (D / 2);
      const int ch = lane * VPL;
      if constexpr (VPL == 2) {
        codes[is_k ? k_byte(ch, D) : v_byte(ch, D)] = (uint8_t)code;
      } else if constexpr (VPL == 4) {
        *reinterpret_cast<uint16_t*>(codes + (is_k ? k_byte(ch, D) : v_byte(ch, D))) = (uint16_t)code;
      } else if (is_k) {
        *reinterpret_cast<uint32_t*>(codes + k_byte(ch, D)) = code;
      } else {
        *reinterpret_cast<uint16_t*>(codes + v_byte(ch, D)) = (uint16_t)code;
        *reinterpret_cast<uint16_t*>(codes + v_byte(ch + 4, D)) = (uint16_t)(code >> 16);
      }
      if (lane % LANES == 0)
        *reinterpret_cast<float2*>(tile + (is_k ? k_params_at(D) : v_params_at(D, NG)) +
                                   ((lane / LANES) * kTile + row) * 8) = make_float2(scale, mn);
    }
  }
}

// Rows read back: code * scale + min, rounded after the product and after the
// sum; a slot below zero gives zeros.  A warp takes HB of a row's K and V heads
// (HB as in append_kernel).  Bounded by HBM; 8,100 rows of 8 heads of 128 take 17 us.
template <int VPL, int LANES, int HB>
__global__ void __launch_bounds__(256)
    read_kernel(const uint8_t* __restrict__ cache, const int32_t* __restrict__ slots, int64_t rows,
                int hkv, int bs, int64_t n_slots, float* __restrict__ k, float* __restrict__ v, int* err) {
  constexpr int D = VPL * 32, NG = 32 / LANES, TB = tile_bytes(D, NG);
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, ch = lane * VPL;
  const int nk = (hkv + HB - 1) / HB, per = 2 * nk;
  const int64_t items = rows * per;
  for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items;
       it += (int64_t)gridDim.x * 8) {
    const int64_t t = quot(it, per);
    const int w = (int)(it - t * per);
    const bool is_k = w < nk;
    const int h0 = (is_k ? w : w - nk) * HB;
    const int64_t slot = slots[t];
    const bool there = slot >= 0 && slot < n_slots;
    if (slot >= n_slots && lane == 0 && err) atomicExch(err, 4);
    uint32_t code[HB] = {};
    float2 p[HB] = {};
    if (there) {
      const uint32_t blk = (uint32_t)slot / (uint32_t)bs, in_blk = (uint32_t)slot - blk * (uint32_t)bs;
      const int row = in_blk % kTile, tiles = bs / kTile;
      const uint8_t* tile = cache + (((int64_t)blk * hkv + h0) * tiles + in_blk / kTile) * TB;
#pragma unroll
      for (int i = 0; i < HB; ++i, tile += (int64_t)tiles * TB) {
        if (HB > 1 && h0 + i >= hkv) break;
        const uint8_t* codes = tile + (is_k ? 0 : v_codes_at(D)) + row * (D / 2);
        if constexpr (VPL == 2) {
          code[i] = codes[is_k ? k_byte(ch, D) : v_byte(ch, D)];
        } else if constexpr (VPL == 4) {
          code[i] = *reinterpret_cast<const uint16_t*>(codes + (is_k ? k_byte(ch, D) : v_byte(ch, D)));
        } else if (is_k) {
          code[i] = *reinterpret_cast<const uint32_t*>(codes + k_byte(ch, D));
        } else {
          code[i] = *reinterpret_cast<const uint16_t*>(codes + v_byte(ch, D)) |
                    (uint32_t)*reinterpret_cast<const uint16_t*>(codes + v_byte(ch + 4, D)) << 16;
        }
        p[i] = *reinterpret_cast<const float2*>(tile + (is_k ? k_params_at(D) : v_params_at(D, NG)) +
                                                ((lane / LANES) * kTile + row) * 8);
      }
    }
    float* dst = (is_k ? k : v) + (t * hkv + h0) * D + ch;
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      if (HB > 1 && h0 + i >= hkv) break;
      float x[VPL];
#pragma unroll
      for (int e = 0; e < VPL; ++e) x[e] = __fadd_rn(__fmul_rn((float)((code[i] >> (4 * e)) & 15u), p[i].x), p[i].y);
      store_row<VPL>(dst + i * D, x);
    }
  }
}

unsigned warp_grid(int64_t items) {
  const int64_t most = (int64_t)ctx()->num_sms * 8;
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, (items + 7) / 8));
}

// Warps that are resident at once; with fewer items a warp takes one head.
int64_t all_warps() { return (int64_t)ctx()->num_sms * 64; }

struct AppendArgs {
  const float *q;
  float* q_out;
  int h;
  const float *k, *v;
  int64_t rows;
  const int32_t *slots, *positions;
  const float *cos_t, *sin_t;
  int64_t max_seq;
  uint8_t* cache;
  Shape s;
};

template <int VPL, int LANES>
int run_append(const AppendArgs& a, cudaStream_t st) {
  const bool few = a.rows * (a.h + 2 * a.s.hkv) <= all_warps();
  const int hb = few ? 1 : 4;
  const int64_t items = a.rows * ((a.h + hb - 1) / hb + 2 * ((a.s.hkv + hb - 1) / hb));
  auto kern = few ? append_kernel<VPL, LANES, 1> : append_kernel<VPL, LANES, 4>;
  return launch(kern, dim3(warp_grid(items)), 256, 0, st, 1, a.q, a.q_out, a.h, a.k, a.v, a.rows, a.slots,
                a.positions, a.cos_t, a.sin_t, a.max_seq, a.cache, a.s.hkv, a.s.bs, a.s.n_blocks * a.s.bs,
                ctx()->dev_err);
}

template <int VPL, int LANES>
int run_read(const Shape& s, const uint8_t* cache, const int32_t* slots, int64_t rows, float* k, float* v,
             cudaStream_t st) {
  const bool few = rows * 2 * s.hkv <= all_warps();
  const int hb = few ? 1 : 4;
  auto kern = few ? read_kernel<VPL, LANES, 1> : read_kernel<VPL, LANES, 4>;
  return launch(kern, dim3(warp_grid(rows * 2 * ((s.hkv + hb - 1) / hb))), 256, 0, st, 1, cache, slots, rows,
                s.hkv, s.bs, s.n_blocks * s.bs, k, v, ctx()->dev_err);
}

// f<VPL, LANES>(...) of a cache's head dim and group.
#define NIMF_KV4_BY_SHAPE(f, s, ...)                                          \
  switch ((s).d * 16 + (s).d / (s).group) {                                   \
    case 64 * 16 + 1: return f<2, 32>(__VA_ARGS__);                           \
    case 64 * 16 + 2: return f<2, 16>(__VA_ARGS__);                           \
    case 128 * 16 + 1: return f<4, 32>(__VA_ARGS__);                          \
    case 128 * 16 + 2: return f<4, 16>(__VA_ARGS__);                          \
    case 128 * 16 + 4: return f<4, 8>(__VA_ARGS__);                           \
    case 256 * 16 + 2: return f<8, 16>(__VA_ARGS__);                          \
    case 256 * 16 + 4: return f<8, 8>(__VA_ARGS__);                           \
    default: return f<8, 4>(__VA_ARGS__);                                     \
  }
int append_by_shape(const AppendArgs& a, cudaStream_t st) { NIMF_KV4_BY_SHAPE(run_append, a.s, a, st) }
int read_by_shape(const Shape& s, const uint8_t* cache, const int32_t* slots, int64_t rows, float* k,
                  float* v, cudaStream_t st) {
  NIMF_KV4_BY_SHAPE(run_read, s, s, cache, slots, rows, k, v, st)
}
#undef NIMF_KV4_BY_SHAPE

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace
}  // namespace kv4
}  // namespace nimf

using namespace nimf;

extern "C" {

int nimf_kv4_cache_bytes(const nimf_kv4_desc* desc, int64_t* bytes) {
  kv4::Shape s;
  NIMF_TRY(kv4::check_desc(desc, "kv4_cache_bytes", &s));
  if (!bytes) return set_error(NIMF_ERR_ARG, "kv4_cache_bytes: NULL result");
  *bytes = s.n_blocks * s.hkv * (s.bs / kv4::kTile) * kv4::tile_bytes(s.d, s.d / s.group);
  return NIMF_OK;
}

int nimf_kv4_reserve_dev(const nimf_kv4_desc* desc, int64_t n_seqs, int64_t max_blocks,
                         const int32_t* n_new, const int32_t* lens, int32_t* lens_out,
                         int32_t* block_table, const int32_t* free_blocks, const int32_t* n_free,
                         int32_t* n_free_out, int64_t max_rows, int32_t* cu_rows, int32_t* slots,
                         int32_t* positions, int32_t* granted, void* stream) {
  cudaStream_t st;
  kv4::Shape s;
  NIMF_TRY(kv4::check_desc(desc, "kv4_reserve", &s));
  if (n_seqs < 0 || n_seqs > kv4::kMaxSeqs || max_blocks < 1 || max_blocks > INT32_MAX / s.bs ||
      max_rows < 0 || max_rows > INT32_MAX)
    return set_error(NIMF_ERR_SHAPE, "kv4_reserve: n_seqs %lld max_blocks %lld max_rows %lld",
                     (long long)n_seqs, (long long)max_blocks, (long long)max_rows);
  if (!free_blocks || !n_free || !n_free_out || !cu_rows ||
      (n_seqs > 0 && (!n_new || !lens || !lens_out || !block_table || !granted)) ||
      (max_rows > 0 && (!slots || !positions)))
    return set_error(NIMF_ERR_ARG, "kv4_reserve: NULL buffer");
  NIMF_TRY(kv4::stream_of(stream, &st));
  kv4::Blocks blocks;
  blocks.bs = (uint32_t)s.bs;
  blocks.magic = (((uint64_t)1 << 36) + s.bs / 16 - 1) / (s.bs / 16);
  const bool own = max_rows <= kv4::kOwnRows || n_seqs == 0;
  // as many threads as requests or warps' rows ask for: scans of few warps are short
  const int64_t want = own ? std::max<int64_t>(n_seqs, max_rows / 4) : kv4::kPoolThreads;
  const unsigned threads = want <= 128 ? 128 : want <= 256 ? 256 : want <= 512 ? 512 : kv4::kPoolThreads;
  NIMF_TRY(kv4::launch(kv4::reserve_kernel, dim3(1), threads, 0, st, 1, (int)n_seqs, max_blocks, blocks, s.n_blocks,
                       n_new, lens, lens_out, block_table, free_blocks, n_free, n_free_out, max_rows, cu_rows,
                       slots, positions, granted, own ? 1 : 0));
  if (own) return NIMF_OK;
  return kv4::launch(kv4::rows_kernel, dim3(kv4::warp_grid((max_rows + 127) / 128)), 256, 0, st, 1, (int)n_seqs,
                     max_blocks, blocks, s.n_blocks, (const int32_t*)lens_out, (const int32_t*)block_table, max_rows,
                     (const int32_t*)cu_rows, (const int32_t*)granted, slots, positions);
}

int nimf_kv4_release_dev(const nimf_kv4_desc* desc, int64_t n_seqs, int64_t max_blocks,
                         const int32_t* finished, int32_t* lens, const int32_t* block_table,
                         int32_t* free_blocks, int32_t* n_free, void* stream) {
  cudaStream_t st;
  kv4::Shape s;
  NIMF_TRY(kv4::check_desc(desc, "kv4_release", &s));
  if (n_seqs < 0 || n_seqs > kv4::kMaxSeqs || max_blocks < 1 || max_blocks > INT32_MAX / s.bs)
    return set_error(NIMF_ERR_SHAPE, "kv4_release: n_seqs %lld max_blocks %lld", (long long)n_seqs,
                     (long long)max_blocks);
  if (n_seqs == 0) return NIMF_OK;
  if (!finished || !lens || !block_table || !free_blocks || !n_free)
    return set_error(NIMF_ERR_ARG, "kv4_release: NULL buffer");
  NIMF_TRY(kv4::stream_of(stream, &st));
  return kv4::launch(kv4::release_kernel, dim3(1), kv4::kPoolThreads, 0, st, 1, n_seqs, max_blocks,
                     s.bs, s.n_blocks, finished, lens, block_table, free_blocks, n_free,
                     ctx()->dev_err);
}

int nimf_kv4_append_dev(const nimf_kv4_desc* desc, void* cache, const float* k, const float* v,
                        int64_t rows, const int32_t* slots, const float* q, float* q_out,
                        int64_t n_heads, const int32_t* positions, const float* cos_t,
                        const float* sin_t, int64_t max_seq, void* stream) {
  cudaStream_t st;
  kv4::Shape s;
  NIMF_TRY(kv4::check_desc(desc, "kv4_append", &s));
  if (rows < 0 || rows > INT32_MAX || n_heads < 0 || n_heads > 65535)
    return set_error(NIMF_ERR_SHAPE, "kv4_append: rows %lld n_heads %lld", (long long)rows,
                     (long long)n_heads);
  if (!cos_t != !sin_t || !q != !q_out || (q && n_heads < 1) || (cos_t && (!positions || max_seq < 1)))
    return set_error(NIMF_ERR_ARG,
                     "kv4_append: cos_t and sin_t come together, with positions and max_seq; q with "
                     "q_out and n_heads");
  if (rows == 0) return NIMF_OK;
  if (!cache || !k || !v || !slots) return set_error(NIMF_ERR_ARG, "kv4_append: NULL buffer");
  for (const void* p : {(const void*)cache, (const void*)k, (const void*)v, (const void*)q,
                        (const void*)q_out, (const void*)cos_t, (const void*)sin_t})
    if (!kv4::aligned(p, 16))
      return set_error(NIMF_ERR_ARG, "kv4_append: buffers must be 16-byte aligned");
  NIMF_TRY(kv4::stream_of(stream, &st));
  return kv4::append_by_shape({q, q_out, q ? (int)n_heads : 0, k, v, rows, slots, positions, cos_t, sin_t,
                               max_seq, (uint8_t*)cache, s}, st);
}

int nimf_kv4_read_dev(const nimf_kv4_desc* desc, const void* cache, const int32_t* slots,
                      int64_t rows, float* k, float* v, void* stream) {
  cudaStream_t st;
  kv4::Shape s;
  NIMF_TRY(kv4::check_desc(desc, "kv4_read", &s));
  if (rows < 0 || rows > INT32_MAX)
    return set_error(NIMF_ERR_SHAPE, "kv4_read: rows %lld", (long long)rows);
  if (rows == 0) return NIMF_OK;
  if (!cache || !slots || !k || !v) return set_error(NIMF_ERR_ARG, "kv4_read: NULL buffer");
  if (!kv4::aligned(cache, 16) || !kv4::aligned(k, 16) || !kv4::aligned(v, 16))
    return set_error(NIMF_ERR_ARG, "kv4_read: buffers must be 16-byte aligned");
  NIMF_TRY(kv4::stream_of(stream, &st));
  return kv4::read_by_shape(s, (const uint8_t*)cache, slots, rows, k, v, st);
}

}  // extern "C"
