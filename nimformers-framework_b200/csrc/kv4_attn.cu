// kv4_attn.cu -- attention of new tokens over the 4-bit paged KV cache.
//
//   out[t][h] = sum_j p_j v^_j / sum_j p_j,  p_j = exp(scale * q . k^_j),
//   k^_j = c_j s_j + m_j per group of channels (v^ likewise),
// over the cached tokens j that row t may see (causal).
//
// The products run on the tensor cores with codes centred at 8: a nibble masked
// into the fp16 number 1024 + c (or 1024 + 16 c for the nibble above it) less
// 1032 (1152) is c - 8 (16 times that) exactly, so eight codes cost nine
// operations.  Scale and minimum enter outside:
//   q . k^_j = sum_groups s_j (q . (c_j - 8)) + (m_j + 8 s_j) sum(q)
//   sum_j p_j v^_j = sum_j (p_j s_j) (c_j - 8) + sum_j p_j (m_j + 8 s_j)
// Centred, both sums of the second line are as small as the result; the codes
// taken from 0 make them grow with the context while the result shrinks, and
// the difference lost 2^-11 of it at 131,000 tokens.
// q and p s are given as two fp16 terms each, high terms in rows 0..7 of the
// MMA's A operand and low terms in rows 8..15, so one 16-row tile carries 8
// query rows at float32's accuracy; both halves of an accumulator are added in
// registers.  The tensor core cuts what an addition shifts out.  So q's high
// terms are integers of 11 bits: their products with the codes and all sums of
// them are exact.  p s, whose values differ by many powers of two, has 22 bits
// of each value, and sums of 32 tokens at most run in the tensor core.
#include <cfloat>

#include "kv4.cuh"

namespace nimf {
namespace kv4 {

namespace {

constexpr int kUnit = 32;        // tokens a warp takes at a time (two tiles)
constexpr int kStages = 2;       // units in flight per warp
constexpr int kRows = 8;         // query rows of a row tile
// Warps of a CTA: with the ring of a 256-channel tile, six fill the shared memory.
__host__ __device__ constexpr int warps_of(int d) { return d <= 128 ? 8 : 6; }

// One CTA's share that begins inside a segment; written for the join.
struct SegInfo {
  int64_t u0, u1;   // the segment's units; u0 < 0: this CTA starts no join
  int32_t b, kvh, tile, pad;
};
struct WsHead {
  int64_t units, ctas;
};
constexpr int kWsHeadBytes = 64;

__host__ __device__ constexpr int part_floats(int d) { return kRows * (d + 2); }

// Rings, then one kept piece per warp.
constexpr int attn_smem(int d, int ng) {
  return warps_of(d) * (kStages * 2 * tile_bytes(d, ng) + part_floats(d) * 4);
}

size_t ws_bytes(int ctas, int d) {
  return kWsHeadBytes + (size_t)ctas * sizeof(SegInfo) + (size_t)ctas * 2 * part_floats(d) * 4;
}

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
  if (a.cu_rows) {
    s.row0 = min((int64_t)max(a.cu_rows[b], 0), a.rows);
    e = min((int64_t)max(a.cu_rows[b + 1], 0), a.rows);
  } else {
    s.row0 = min(b, a.rows);
    e = min(b + 1, a.rows);
  }
  s.n = (int)max(e - s.row0, (int64_t)0);
  s.len = (int)min((int64_t)max(a.lens[b], 0), a.width * a.bs);
  return s;
}
__device__ __forceinline__ int seq_units(int len) { return max(1, (len + kUnit - 1) / kUnit); }
__device__ __forceinline__ int seq_tiles(int n, int r) {
  return (int)(((int64_t)n * r + kRows - 1) / kRows);
}

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
// Two floats as fp16 high terms and the fp16 rests.
__device__ __forceinline__ void split_f16x2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x0, x1);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x0 - f.x, x1 - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
// Two floats up to 2^11 as integers and fp16 rests, both times f.
__device__ __forceinline__ void split_int(float x0, float x1, float f, uint32_t& hi, uint32_t& lo) {
  const float r0 = rintf(x0), r1 = rintf(x1);
  const __half2 h = __floats2half2_rn(r0 * f, r1 * f), l = __floats2half2_rn((x0 - r0) * f, (x1 - r1) * f);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
// The codes of the even (odd: 16 times them) nibbles of the low and the third
// byte's half words, less 8, as two fp16 numbers.
__device__ __forceinline__ uint32_t codes_f16(uint32_t w, bool odd) {
  uint32_t v = lop3_and_or(w, odd ? 0x00F000F0u : 0x000F000Fu, 0x64006400u), r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(odd ? 0xE480E480u : 0xE408E408u));
  return r;
}
// 2^(e - 127) for an exponent field e clamped to the normal range.
__device__ __forceinline__ float pow2_field(int e) {
  return __int_as_float(max(1, min(254, e)) << 23);
}
__device__ __forceinline__ int exp_field(float x) { return (__float_as_int(x) >> 23) & 255; }

// N consecutive words of shared memory.
template <int N>
__device__ __forceinline__ void lds(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x;
    w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x;
      w[4 * i + 1] = v.y;
      w[4 * i + 2] = v.z;
      w[4 * i + 3] = v.w;
    }
  }
}

// Attention of few rows per sequence (decode and short chunks).
//
// Work: a segment is 8 query rows (tokens x heads of one KV head) of one
// sequence over all its tokens; its units are 32 tokens.  All units of all
// segments lie on one line that is cut evenly among the warps of a grid that
// fits the GPU at once, whatever the lengths are.  A warp's pieces of
// segments that other warps continue are joined in shared memory, and pieces
// that other CTAs continue go to the workspace for join_kernel.
//
// Each warp streams its tiles with bulk copies into its own two-stage ring.
template <int D, int NG>
__global__ void __launch_bounds__(warps_of(D) * 32, D <= 128 ? 2 : 1) attn_kernel(const Args a) {
  constexpr int NC = D / 32, NS = D / 64, G = D / NG, W = warps_of(D);
  constexpr int TB = tile_bytes(D, NG), PF = part_floats(D);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[W][kStages];
  __shared__ int64_t sh[33];
  __shared__ int64_t s_start[W + 1];        // the warps' first units
  __shared__ int64_t s_b[W], s_off[W];      // where on the line those are
  __shared__ SegInfo s_seg[W][2];           // kept pieces: at the warp's first unit, at its last
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  griddep_launch_dependents();
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[warp][i], 1);
    mbar_fence_init();
  }
  griddep_wait();

  // ---- the line of units, and where this CTA's warps begin on it
  auto line_units = [&](int64_t b) -> int64_t {
    if (b >= a.n_seqs) return 0;
    const Seq s = seq_of(a, b);
    return (int64_t)seq_units(s.len) * seq_tiles(s.n, a.r) * a.hkv;
  };
  int64_t total = 0;
  for (int64_t b0 = 0; b0 < a.n_seqs; b0 += W * 32) {
    int64_t sum;
    block_scan<int64_t>(line_units(b0 + tid), sh, &sum);
    total += sum;
  }
  const int64_t ctas = max((int64_t)1, min((int64_t)gridDim.x, (total + W - 1) / W));
  const int64_t cta = blockIdx.x;
  SegInfo* info = reinterpret_cast<SegInfo*>(a.ws + kWsHeadBytes);
  float* parts = reinterpret_cast<float*>(a.ws + kWsHeadBytes + (size_t)gridDim.x * sizeof(SegInfo));
  if (cta == 0 && tid == 0) {
    WsHead* hd = reinterpret_cast<WsHead*>(a.ws);
    hd->units = total;
    hd->ctas = ctas;
  }
  if (cta >= ctas || total == 0) {
    if (tid == 0) info[cta].u0 = -1;
    return;
  }
  const int64_t cta_a = cta * total / ctas, cta_b = (cta + 1) * total / ctas;
  if (tid <= W) s_start[tid] = cta_a + tid * (cta_b - cta_a) / W;
  if (tid < W * 2) s_seg[tid >> 1][tid & 1].u0 = -1;
  __syncthreads();
  for (int64_t b0 = 0, base = 0; b0 < a.n_seqs && base < cta_b; b0 += W * 32) {
    const int64_t u = line_units(b0 + tid);
    int64_t sum;
    const int64_t end = base + block_scan<int64_t>(u, sh, &sum);
    for (int w = 0; w < W; ++w)
      if (s_start[w] >= end - u && s_start[w] < end) {
        s_b[w] = b0 + tid;
        s_off[w] = s_start[w] - (end - u);
      }
    base += sum;
  }
  __syncthreads();
  if (tid == 0) {  // the segment cut by this CTA's beginning, joined in its name if it is the first cut
    const int64_t b = s_b[0], off = s_off[0];
    const Seq s = seq_of(a, b);
    const int tiles = seq_tiles(s.n, a.r), nu = seq_units(s.len);
    const int64_t seg = off / nu;
    SegInfo si;
    si.u0 = cta_a - (off - seg * nu);
    si.u1 = si.u0 + nu;
    si.b = (int32_t)b;
    si.kvh = (int32_t)(seg / tiles);
    si.tile = (int32_t)(seg % tiles);
    si.pad = 0;
    if (si.u0 == cta_a || si.u0 < (cta - 1) * total / ctas) si.u0 = -1;
    info[cta] = si;
  }

  const int64_t w_a = s_start[warp], w_b = s_start[warp + 1];
  uint8_t* ring = smem + (size_t)warp * kStages * 2 * TB;
  float* kept = reinterpret_cast<float*>(smem + (size_t)W * kStages * 2 * TB) + warp * PF;
  uint32_t phase = 0;                       // parity of each stage's next use
  int64_t b = 0, off = 0;
  if (w_a < w_b) {
    b = s_b[warp];
    off = s_off[warp];
  }
  for (int64_t at = w_a; at < w_b;) {
    const Seq s = seq_of(a, b);
    const int tiles = seq_tiles(s.n, a.r), nu = seq_units(s.len);
    if (off >= (int64_t)nu * tiles * a.hkv) {  // the next sequence
      off = 0;
      ++b;
      continue;
    }
    const int64_t seg = off / nu;
    const int u_first = (int)(off - seg * nu);
    const int u_count = (int)min((int64_t)(nu - u_first), w_b - at);
    const int kvh = (int)(seg / tiles), tile = (int)(seg - (int64_t)kvh * tiles);

    // this lane's query row (row g of the tile) and how far it sees
    const int rr = tile * kRows + g;
    const bool row_ok = rr < s.n * a.r;
    const int tok = rr / a.r, hq = kvh * a.r + rr - tok * a.r;
    const int limit = row_ok ? max(0, min(s.len, s.len - s.n + tok + 1)) : 0;
    const int last_tok = min(s.n - 1, (tile * kRows + kRows - 1) / a.r);
    const int seg_len = max(0, min(s.len, s.len - s.n + last_tok + 1));  // no row sees further
    const int u_live = min(u_first + u_count, (seg_len + kUnit - 1) / kUnit);

    int32_t blk = 0;                        // the block of tile 2 * ids_at + lane
    int ids_at = -1024;
    auto issue = [&](int u, int stage) -> int {
      if (u - ids_at >= 16) {
        ids_at = u;
        const int64_t t0 = (int64_t)(2 * u + lane) * kTile;
        blk = t0 < seg_len ? a.table[b * a.width + t0 / a.bs] : -1;
        if (blk < 0 || blk >= a.n_blocks) {  // never read: its tokens are left out
          if (t0 < seg_len && a.err) atomicExch(a.err, 4);
          blk = -1;
        }
      }
      const int p0 = __shfl_sync(0xffffffffu, blk, 2 * (u - ids_at));
      const int p1 = __shfl_sync(0xffffffffu, blk, 2 * (u - ids_at) + 1);
      if (lane == 0) {
        const int per = a.bs / kTile;
        mbar_arrive_expect_tx(&full[warp][stage], (p0 >= 0 ? TB : 0) + (p1 >= 0 ? TB : 0));
        uint8_t* dst = ring + stage * 2 * TB;
        if (p0 >= 0)
          bulk_g2s(dst, a.cache + (((int64_t)p0 * a.hkv + kvh) * per + (2 * u) % per) * TB, TB,
                   &full[warp][stage]);
        if (p1 >= 0)
          bulk_g2s(dst + TB, a.cache + (((int64_t)p1 * a.hkv + kvh) * per + (2 * u + 1) % per) * TB,
                   TB, &full[warp][stage]);
      }
      return (p0 >= 0 ? 1 : 0) | (p1 >= 0 ? 2 : 0);
    };

    // which of a stage's tiles are there: two bits a stage.  The stage of a
    // unit follows the ring's position over the warp's whole life.
    uint32_t there = 0;
    for (int i = 0; i < kStages; ++i)
      if (u_first + i < u_live) there |= issue(u_first + i, i) << (2 * i);

    // ---- query fragments: two fp16 terms of q * scale * log2(e) * 2^k
    uint32_t qf[NC][2][4];
    float qsum[NG], row_f;
    {
      float x[NC][8], amax = 0.f;
      const float* qr = a.q + ((s.row0 + tok) * a.h + hq) * D;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        float4 v0 = make_float4(0.f, 0.f, 0.f, 0.f), v1 = v0;
        if (row_ok) {
          v0 = *reinterpret_cast<const float4*>(qr + 32 * j + 8 * c);
          v1 = *reinterpret_cast<const float4*>(qr + 32 * j + 8 * c + 4);
        }
        x[j][0] = v0.x; x[j][1] = v0.y; x[j][2] = v0.z; x[j][3] = v0.w;
        x[j][4] = v1.x; x[j][5] = v1.y; x[j][6] = v1.z; x[j][7] = v1.w;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[j][i] *= a.scale2;
          amax = fmaxf(amax, fabsf(x[j][i]));
        }
      }
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (j * 32 / G == n)
#pragma unroll
            for (int i = 0; i < 8; ++i) t += x[j][i];
        t += __shfl_xor_sync(0xffffffffu, t, 1);
        t += __shfl_xor_sync(0xffffffffu, t, 2);
        qsum[n] = t;
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // the largest magnitude goes to [2^10, 2^11): integers and their rests
      const int e = max(14, min(244, exp_field(amax)));
      const float up = pow2_field(264 - e);
      row_f = pow2_field(e - 10);           // 1 / up
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int p = 0; p < 2; ++p) {       // even nibbles, then odd ones (16 c)
          const float f = p ? 0.0625f : 1.f;
          split_int(x[j][p] * up, x[j][p + 4] * up, f, qf[j][p][0], qf[j][p][1]);
          split_int(x[j][p + 2] * up, x[j][p + 6] * up, f, qf[j][p][2], qf[j][p][3]);
        }
    }

    // ---- online softmax over the units
    float m = -INFINITY, l = 0.f, mins[NG];
    float o[NS][2][4][2];                   // [span][half][nibble][column]
    int e_run = 20;                         // exponent field of the largest value scale so far
#pragma unroll
    for (int n = 0; n < NG; ++n) mins[n] = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][j][k][0] = o[i][j][k][1] = 0.f;

    const int pi = g ^ ((g >> 1) & 1);      // the token of key column g
    bool failed = false;
    for (int u = u_first, st = 0; u < u_live; ++u, st ^= 1) {
      if (!mbar_wait(&full[warp][st], (phase >> st) & 1u)) {
        if (a.err) atomicExch(a.err, 6);
        failed = true;
        break;
      }
      phase ^= 1u << st;
      const uint8_t* buf = ring + st * 2 * TB;
      const uint32_t has = there >> (2 * st);

      // Scores.  Column n of a key tile is token n ^ (n >> 1 & 1): the two
      // columns of a lane stay two neighbouring tokens, and the value rows
      // that the four lanes of a quad read lie in different banks.
      float sc[2][2][2];                    // [tile][8-token half][column]
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t w[NC];
          lds<NC>(buf + t * TB + (hf * 8 + pi) * (D / 2) + c * NC * 4, w);
          float acc[NG][4];
#pragma unroll
          for (int n = 0; n < NG; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            const uint32_t w8 = w[j] >> 8;
            mma_f16_16816(acc[j * 32 / G], qf[j][0][0], qf[j][0][1], qf[j][0][2], qf[j][0][3],
                          codes_f16(w[j], false), codes_f16(w8, false));
            mma_f16_16816(acc[j * 32 / G], qf[j][1][0], qf[j][1][1], qf[j][1][2], qf[j][1][3],
                          codes_f16(w[j], true), codes_f16(w8, true));
          }
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            const float4 p = *reinterpret_cast<const float4*>(
                buf + t * TB + k_params_at(D) + (n * kTile + hf * 8 + 2 * c) * 8);
            const float a0 = (acc[n][0] + acc[n][2]) * row_f, a1 = (acc[n][1] + acc[n][3]) * row_f;
            const float k0 = c & 1 ? p.z : p.x, k1 = c & 1 ? p.x : p.z;
            s0 = fmaf(a0, k0, fmaf(qsum[n], fmaf(8.f, k0, c & 1 ? p.w : p.y), s0));
            s1 = fmaf(a1, k1, fmaf(qsum[n], fmaf(8.f, k1, c & 1 ? p.y : p.w), s1));
          }
          const int t0 = u * kUnit + t * kTile + hf * 8 + 2 * c;
          const bool in = (has >> t) & 1u;
          sc[t][hf][0] = in && t0 + (c & 1) < limit ? s0 : -INFINITY;
          sc[t][hf][1] = in && t0 + 1 - (c & 1) < limit ? s1 : -INFINITY;
        }
      float mu = sc[0][0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mu = fmaxf(mu, sc[i >> 2][(i >> 1) & 1][i & 1]);
      mu = fmaxf(mu, __shfl_xor_sync(0xffffffffu, mu, 1));
      mu = fmaxf(mu, __shfl_xor_sync(0xffffffffu, mu, 2));
      const float m_new = fmaxf(m, mu);
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      const float corr = ex2(m - ref);      // 0 while nothing was seen
      m = m_new;

      // {scale, minimum} of the values of this lane's tokens; tokens past the
      // end and blocks that are not there count as zeros, whatever lies there
      auto v_params = [&](int n, int t, int hf) -> float4 {
        const float4 p = *reinterpret_cast<const float4*>(
            buf + t * TB + v_params_at(D, NG) + (n * kTile + hf * 8 + 2 * c) * 8);
        const int t0 = u * kUnit + t * kTile + hf * 8 + 2 * c;
        const bool in = (has >> t) & 1u;
        const bool ok0 = in && t0 < seg_len, ok1 = in && t0 + 1 < seg_len;
        const float4 q = make_float4(ok0 ? p.x : 0.f, ok0 ? p.y : 0.f, ok1 ? p.z : 0.f, ok1 ? p.w : 0.f);
        return c & 1 ? make_float4(q.z, q.w, q.x, q.y) : q;
      };
      float vmax = 0.f;
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 p = v_params(n, i >> 1, i & 1);
          vmax = fmaxf(vmax, fmaxf(p.x, p.z));
        }
      vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 1));
      vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 2));
      // p * scale goes to the fp16 range by the power of two that brings the
      // largest scale so far to [2^14, 2^15)
      const int e_new = max(e_run, min(254, exp_field(vmax)));
      const float corr_o = e_new - e_run > 126 ? 0.f : corr * pow2_field(127 - (e_new - e_run));
      e_run = e_new;
      const float up = pow2_field(268 - e_run);

      // masked tokens are marked by a negative p
      l *= corr;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p = ex2(sc[t][hf][e] - ref);
            l += p;
            sc[t][hf][e] = sc[t][hf][e] == -INFINITY ? -1.f : p;
          }

      // Values, half a span (32 channels, one group) at a time.  A unit's
      // products are summed apart and then added, so that the tensor core's
      // own accumulation never runs over more than 32 tokens.
      uint32_t pa[2][4];
      uint32_t vw[2][4][NS];                // the rows of this lane's 8 tokens
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = (i >> 1) * 8 + 2 * c + ((i & 1) ^ (c & 1));
          lds<NS>(buf + t * TB + v_codes_at(D) + row * (D / 2) + g * NS * 4, vw[t][i]);
        }
#pragma unroll
      for (int sp = 0; sp < NS; ++sp)
#pragma unroll
        for (int hv = 0; hv < 2; ++hv) {
          const int n = (64 * sp + 32 * hv) / G;
          if ((64 * sp + 32 * hv) % G == 0) {
            mins[n] *= corr;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                const float4 p = v_params(n, t, hf);
                const float p0 = sc[t][hf][0], p1 = sc[t][hf][1];
                const float w0 = p0 < 0.f ? 0.f : p0 * (p.x * up);
                const float w1 = p1 < 0.f ? 0.f : p1 * (p.z * up);
                if (!(p0 < 0.f)) mins[n] = fmaf(p0, fmaf(8.f, p.x, p.y), mins[n]);
                if (!(p1 < 0.f)) mins[n] = fmaf(p1, fmaf(8.f, p.z, p.w), mins[n]);
                split_f16x2(w0, w1, pa[t][2 * hf], pa[t][2 * hf + 1]);
              }
          }
          float acc[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const uint32_t x0 = prmt(vw[t][0][sp], vw[t][1][sp], hv ? 0x7632 : 0x5410);
            const uint32_t x1 = prmt(vw[t][2][sp], vw[t][3][sp], hv ? 0x7632 : 0x5410);
            const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
            mma_f16_16816(acc[0], pa[t][0], pa[t][1], pa[t][2], pa[t][3], codes_f16(x0, false), codes_f16(x1, false));
            mma_f16_16816(acc[1], pa[t][0], pa[t][1], pa[t][2], pa[t][3], codes_f16(x0, true), codes_f16(x1, true));
            mma_f16_16816(acc[2], pa[t][0], pa[t][1], pa[t][2], pa[t][3], codes_f16(y0, false), codes_f16(y1, false));
            mma_f16_16816(acc[3], pa[t][0], pa[t][1], pa[t][2], pa[t][3], codes_f16(y0, true), codes_f16(y1, true));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[sp][hv][i][0] = fmaf(o[sp][hv][i][0], corr_o, acc[i][0] + acc[i][2]);
            o[sp][hv][i][1] = fmaf(o[sp][hv][i][1], corr_o, acc[i][1] + acc[i][3]);
          }
        }
      __syncwarp();                         // the stage's readers are done
      if (u + kStages < u_live)
        there = (there & ~(3u << (2 * st))) | (uint32_t)issue(u + kStages, st) << (2 * st);
    }
    if (failed) {  // the copies still in flight, then out; the answer is not valid
      for (int st = 0; st < kStages; ++st) (void)mbar_wait(&full[warp][st], (phase >> st) & 1u);
      break;
    }

    // ---- the piece's sums, in real units
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      mins[n] += __shfl_xor_sync(0xffffffffu, mins[n], 1);
      mins[n] += __shfl_xor_sync(0xffffffffu, mins[n], 2);
    }
    const float f_even = pow2_field(e_run - 14), f_odd = pow2_field(e_run - 18);
    const bool whole = u_count == nu;
    const int64_t u0 = at - u_first;
    const int k = u0 <= w_a ? 0 : 1;
    // a piece at the warp's last unit lies in the ring, whose copies are all read
    float* piece = k ? reinterpret_cast<float*>(ring) : kept;
    float* dst = whole ? a.out + ((s.row0 + tok) * a.h + hq) * D : piece + g * D;
    const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
    if (row_ok || !whole)
#pragma unroll
      for (int sp = 0; sp < NS; ++sp)
#pragma unroll
        for (int hv = 0; hv < 2; ++hv) {
          const float mn = mins[(64 * sp + 32 * hv) / G];
          float r8[8];
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              r8[4 * e + i] = fmaf(o[sp][hv][i][e], i & 1 ? f_odd : f_even, mn) * inv;
          float4* p4 = reinterpret_cast<float4*>(dst + 64 * sp + 32 * hv + 8 * c);
          p4[0] = make_float4(r8[0], r8[1], r8[2], r8[3]);
          p4[1] = make_float4(r8[4], r8[5], r8[6], r8[7]);
        }
    if (!whole) {
      if (c == 0) {
        piece[kRows * D + g] = m;
        piece[kRows * D + kRows + g] = l;
      }
      if (lane == 0) {
        SegInfo& si = s_seg[warp][k];
        si.u0 = u0;
        si.u1 = u0 + nu;
        si.b = (int32_t)b;
        si.kvh = kvh;
        si.tile = tile;
      }
    }
    at += u_count;
    off += u_count;
  }

  // ---- pieces of one segment in neighbouring warps
  __syncthreads();
  auto piece_at = [&](int i) -> const float* {
    return i & 1 ? reinterpret_cast<const float*>(smem + (size_t)(i >> 1) * kStages * 2 * TB)
                 : reinterpret_cast<const float*>(smem + (size_t)W * kStages * 2 * TB) + (i >> 1) * PF;
  };
  for (int i = 0; i < 2 * W;) {
    const SegInfo si = s_seg[i >> 1][i & 1];
    if (si.u0 < 0) {
      ++i;
      continue;
    }
    int end = i + 1;
    while (end < 2 * W && (s_seg[end >> 1][end & 1].u0 < 0 || s_seg[end >> 1][end & 1].u0 == si.u0)) ++end;
    const bool whole = si.u0 >= cta_a && si.u1 <= cta_b;
    const Seq s = seq_of(a, si.b);
    float* slot = parts + (size_t)(2 * cta + (si.u0 <= cta_a ? 0 : 1)) * PF;
    for (int x = tid; x < kRows * D; x += W * 32) {
      const int row = x / D, d = x - row * D;
      float M = -INFINITY;
      for (int j = i; j < end; ++j)
        if (s_seg[j >> 1][j & 1].u0 >= 0) M = fmaxf(M, piece_at(j)[kRows * D + row]);
      const float ref = M == -INFINITY ? 0.f : M;
      float L = 0.f, acc = 0.f;
      for (int j = i; j < end; ++j)
        if (s_seg[j >> 1][j & 1].u0 >= 0) {
          const float* p = piece_at(j);
          const float f = ex2(p[kRows * D + row] - ref);
          L = fmaf(f, p[kRows * D + kRows + row], L);
          acc = fmaf(f, p[x], acc);
        }
      if (whole) {
        const int rr = si.tile * kRows + row;
        if (rr < s.n * a.r) {
          const int tok = rr / a.r, hq = si.kvh * a.r + rr - tok * a.r;
          a.out[((s.row0 + tok) * a.h + hq) * D + d] = L == 0.f ? 0.f : acc / L;
        }
      } else {
        slot[x] = acc;
        if (d == 0) {
          slot[kRows * D + row] = M;
          slot[kRows * D + kRows + row] = L;
        }
      }
    }
    i = end;
  }
}

// Joins the segments that several CTAs share.  Block (i, row): the segment
// that CTA i's beginning cuts, if that is the segment's first cut.  Its parts
// are taken in the order of the CTAs, so the result does not depend on timing.
constexpr int kJoinThreads = 256;
template <int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Args a) {
  constexpr int PF = part_floats(D), GR = kJoinThreads / D;
  extern __shared__ __align__(16) float wgt[];  // one weight per part
  __shared__ float red[kJoinThreads];
  __shared__ float s_m[32], s_l[32];
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x, row = blockIdx.y;
  const int64_t cta = blockIdx.x;
  const SegInfo* info = reinterpret_cast<const SegInfo*>(a.ws + kWsHeadBytes);
  const float* parts = reinterpret_cast<const float*>(a.ws + kWsHeadBytes + (size_t)gridDim.x * sizeof(SegInfo));
  const SegInfo si = info[cta];
  if (si.u0 < 0) return;
  const Seq s = seq_of(a, si.b);
  const int rr = si.tile * kRows + row;
  if (rr >= s.n * a.r) return;
  const WsHead hd = *reinterpret_cast<const WsHead*>(a.ws);
  // the segment's parts: CTA cta - 1, then cta .. up to the one that holds its end
  const int64_t last = (si.u1 - 1) * hd.ctas / hd.units;  // a first guess, put right below
  int64_t hi = last;
  while (hi + 1 < hd.ctas && (hi + 1) * hd.units / hd.ctas < si.u1) ++hi;
  while (hi * hd.units / hd.ctas >= si.u1) --hi;
  const int n = (int)(hi - (cta - 1) + 1);
  auto part = [&](int j) -> const float* {
    const int64_t x = cta - 1 + j;
    const bool second = j == 0 && si.u0 > x * hd.units / hd.ctas;
    return parts + (size_t)(2 * x + (second ? 1 : 0)) * PF;
  };
  float M = -INFINITY;
  for (int j = tid; j < n; j += kJoinThreads) M = fmaxf(M, part(j)[kRows * D + row]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((tid & 31) == 0) s_m[tid >> 5] = M;
  __syncthreads();
  M = s_m[0];
  for (int i = 1; i < kJoinThreads / 32; ++i) M = fmaxf(M, s_m[i]);
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  for (int j = tid; j < n; j += kJoinThreads) {
    const float* p = part(j);
    const float f = ex2(p[kRows * D + row] - ref);
    wgt[j] = f;
    L = fmaf(f, p[kRows * D + kRows + row], L);
  }
  L = warp_sum(L);
  if ((tid & 31) == 0) s_l[tid >> 5] = L;
  __syncthreads();
  L = 0.f;
  for (int i = 0; i < kJoinThreads / 32; ++i) L += s_l[i];
  const int d = tid % D, gr = tid / D;
  float acc = 0.f;
#pragma unroll 4
  for (int j = gr; j < n; j += GR) acc = fmaf(wgt[j], part(j)[row * D + d], acc);
  if (GR > 1) {
    red[tid] = acc;
    __syncthreads();
    if (gr == 0)
      for (int i = 1; i < GR; ++i) acc += red[i * D + d];
  }
  if (gr == 0) {
    const int tok = rr / a.r, hq = si.kvh * a.r + rr - tok * a.r;
    a.out[((s.row0 + tok) * a.h + hq) * D + d] = L == 0.f ? 0.f : acc / L;
  }
}

int grid_of(int d) {
  Context* c = ctx();
  return (c ? c->num_sms : 148) * (d <= 128 ? 2 : 1);
}

template <int D, int NG>
int run_attn(const Args& a, cudaStream_t st) {
  const int smem = attn_smem(D, NG);
  NIMF_TRY(allow_smem((const void*)attn_kernel<D, NG>, smem));
  const int ctas = grid_of(D);
  NIMF_TRY(launch(attn_kernel<D, NG>, dim3(ctas), warps_of(D) * 32, smem, st, 1, a));
  return launch(join_kernel<D>, dim3(ctas, kRows), kJoinThreads, (size_t)ctas * 4, st, 1, a);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace kv4
}  // namespace nimf

using namespace nimf;

extern "C" {

int nimf_kv4_attention_workspace(const nimf_kv4_desc* desc, int64_t n_heads, int64_t* bytes) {
  kv4::Shape s;
  Context* c;
  NIMF_TRY(kv4::check_desc(desc, "kv4_attention_workspace", &s));
  if (n_heads < 1 || n_heads % s.hkv)
    return set_error(NIMF_ERR_SHAPE, "kv4_attention_workspace: n_heads %lld is no multiple of n_kv_heads %d",
                     (long long)n_heads, s.hkv);
  if (!bytes) return set_error(NIMF_ERR_ARG, "kv4_attention_workspace: NULL result");
  NIMF_TRY(require_ctx(&c));
  *bytes = (int64_t)kv4::ws_bytes(kv4::grid_of(s.d), s.d);
  return NIMF_OK;
}

int nimf_kv4_attention_dev(const nimf_kv4_desc* desc, const void* cache, const float* q,
                           int64_t rows, int64_t n_heads, int64_t n_seqs, const int32_t* cu_rows,
                           const int32_t* lens, const int32_t* block_table, int64_t max_blocks,
                           int64_t max_new, float scale, float* out, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  cudaStream_t st;
  kv4::Shape s;
  NIMF_TRY(kv4::check_desc(desc, "kv4_attention", &s));
  if (rows < 0 || rows > INT32_MAX || n_heads < 1 || n_heads % s.hkv || n_heads > 65535 ||
      n_seqs < 0 || n_seqs > INT32_MAX || max_blocks < 1 || max_blocks > INT32_MAX / s.bs || max_new < 0)
    return set_error(NIMF_ERR_SHAPE,
                     "kv4_attention: rows %lld n_heads %lld (a multiple of n_kv_heads %d) n_seqs "
                     "%lld max_blocks %lld max_new %lld",
                     (long long)rows, (long long)n_heads, s.hkv, (long long)n_seqs,
                     (long long)max_blocks, (long long)max_new);
  if (rows == 0 || n_seqs == 0) return NIMF_OK;
  if (!cache || !q || !lens || !block_table || !out || !workspace)
    return set_error(NIMF_ERR_ARG, "kv4_attention: NULL buffer");
  if (!kv4::aligned16(cache) || !kv4::aligned16(q) || !kv4::aligned16(out) || !kv4::aligned16(workspace))
    return set_error(NIMF_ERR_ARG, "kv4_attention: buffers must be 16-byte aligned");
  NIMF_TRY(kv4::stream_of(stream, &st));
  if (workspace_bytes < (int64_t)kv4::ws_bytes(kv4::grid_of(s.d), s.d))
    return set_error(NIMF_ERR_ARG, "kv4_attention: %lld bytes of workspace, nimf_kv4_attention_workspace asks for %lld",
                     (long long)workspace_bytes, (long long)kv4::ws_bytes(kv4::grid_of(s.d), s.d));
  kv4::Args a = {};
  a.cache = (const uint8_t*)cache;
  a.q = q;
  a.cu_rows = cu_rows;
  a.lens = lens;
  a.table = block_table;
  a.out = out;
  a.ws = (unsigned char*)workspace;
  a.err = ctx()->dev_err;
  a.n_seqs = n_seqs;
  a.rows = rows;
  a.width = max_blocks;
  a.n_blocks = s.n_blocks;
  a.h = (int)n_heads;
  a.hkv = s.hkv;
  a.r = (int)(n_heads / s.hkv);
  a.bs = s.bs;
  a.scale2 = (float)((double)scale * 1.4426950408889634);
  switch (s.d * 16 + s.d / s.group) {
    case 64 * 16 + 1: return kv4::run_attn<64, 1>(a, st);
    case 64 * 16 + 2: return kv4::run_attn<64, 2>(a, st);
    case 128 * 16 + 1: return kv4::run_attn<128, 1>(a, st);
    case 128 * 16 + 2: return kv4::run_attn<128, 2>(a, st);
    case 128 * 16 + 4: return kv4::run_attn<128, 4>(a, st);
    case 256 * 16 + 2: return kv4::run_attn<256, 2>(a, st);
    case 256 * 16 + 4: return kv4::run_attn<256, 4>(a, st);
    default: return kv4::run_attn<256, 8>(a, st);
  }
}

}  // extern "C"
