// kv4_attn.cu -- attention of new tokens over the 4-bit paged KV cache.
//
//   out[t][h] = sum_j p_j v^_j / sum_j p_j,  p_j = exp(scale * q . k^_j),
//   k^_j = c_j s_j + m_j per group of channels (v^ likewise),
// over the cached tokens j that row t may see (causal).
//
// The products run on the tensor cores with the codes as they are: a nibble
// masked in place in a 16-bit lane IS the fp16 number c * 2^-24 (a subnormal,
// or 16 c * 2^-24 for the nibble above it), so eight codes cost five logic
// operations and nothing is converted.  Scale and minimum enter outside:
//   q . k^_j = sum_groups s_j (q . (c_j - 8)) + (m_j + 8 s_j) sum(q)
//   sum_j p_j v^_j = sum_j w_j (c_j - 8) + sum_j p_j (m_j + 8 s_j),  w_j = p_j s_j
// The codes count from 8, so that the sums are as small as the result: counted
// from 0 they grow with the context while the result shrinks, and their
// difference lost 2^-11 of it at 131,000 tokens.  The 8 is taken off in the
// accumulators' first value: -8 sum(q), and -8 sum(w) out of one MMA.
//
// The codes are the A operand (16 tokens, or 16 channels of the values), q and
// w the B operand: 4 query rows a tile, each as two columns, an integer that
// fp16 holds and the fp16 rest of it.  The tensor core cuts what an addition shifts
// out; sums of the integer columns stay below 2^24 and are exact, the rests
// are small, and so products and sums have float32's accuracy.
// q's integers are as large as those sums allow: a row's magnitudes add up to
// 2^20 at most and none reaches 2^15 (fp16's end, with room for a rounding), so a
// channel is off by 2^-22 of itself, or by 2^-13 of an integer's step where that is
// more: 2^-27 of a row's largest channel if that one stands out (with 11 bits for
// the largest it was 2^-23, and a channel a hundred times the others cost these
// more than float32's sums do).  w's integers, of 11 bits, count from the largest w
// of the 32 tokens of a unit, 2^-23 of which is nothing to their sum.
//
// Times are those of captured calls over two sets of buffers in turn.
// Long contexts are bounded by HBM and by the ALU that masks the nibbles: 4
// requests of 65,537 to 131,000 tokens and 8 KV heads of 128 take 91 us, 5.2 TB/s
// (102 us, 4.6 TB/s, where every call has buffers of its own).
// Short calls are latency, from the plan to the join: 64 ragged requests up to
// 4,096 tokens 22.4 us (16 heads of 256 over 4: 29), one of 519 tokens with 32 KV
// heads 9.9 us.
#include <algorithm>
#include <cfloat>

#include "kv4.cuh"

namespace nimf {
namespace kv4 {

namespace {

constexpr int kUnit = 32;        // tokens a warp takes at a time (two tiles)
constexpr int kStages = 2;       // units in flight per warp
// Warps of a CTA, CTAs of an SM.  16 warps with 128 registers a thread fill an
// SM: in one CTA where their rings fit its shared memory, so that more of a
// segment is joined there, else in two.  More rows a segment need twice the
// registers; with the ring of a 256-channel tile six warps fill the shared memory.
__host__ __device__ constexpr int warps_of(int d, int ng, int nb) {
  return d > 128 ? 6 : nb == 1 && ng <= 2 ? 16 : 8;
}
__host__ __device__ constexpr int ctas_per_sm(int d, int ng, int nb) { return d <= 128 && nb == 1 && ng > 2 ? 2 : 1; }

// A kept piece of a segment, and (in the workspace) the segment that a CTA's
// beginning cuts first: u0 its first unit on the line, -1 for none.
struct SegInfo {
  int64_t u0, u1;
  int64_t row0;     // the sequence's first row
  int32_t n;        // and its rows
  int32_t kvh, tile;
  int32_t parts;    // join: CTAs that hold a part, counted from the one before
  int32_t second;   // join: the first of them holds it as its last segment
};

// What a CTA's end needs to know of its part of the line: how CTAs' parts are
// cut, its own [begin, end), where it begins (unit off of sequence b), CTAs in
// use.  It lies in shared memory: in registers it cost spills in the main loop.
struct Line {
  int64_t each, more, begin, end, off, b, ctas;
};

// A segment's query rows: 4 per column tile of the MMA's B operand.
__host__ __device__ constexpr int rows_of(int nb) { return 4 * nb; }
constexpr int kMaxNB = 4;
__host__ __device__ constexpr int part_floats(int d, int nb) { return rows_of(nb) * (d + 2); }

// Rings, then one kept piece per warp.
constexpr int attn_smem(int d, int ng, int nb) {
  return warps_of(d, ng, nb) * (kStages * 2 * tile_bytes(d, ng) + part_floats(d, nb) * 4);
}

size_t ws_bytes(int ctas, int d) {
  return (size_t)ctas * sizeof(SegInfo) + (size_t)ctas * 2 * part_floats(d, kMaxNB) * 4;
}

__device__ __forceinline__ int seq_units(int len) { return max(1, (len + kUnit - 1) / kUnit); }
template <int ROWS>
__device__ __forceinline__ int seq_tiles(int n, int r) {
  return (int)(((int64_t)n * r + ROWS - 1) / ROWS);
}

// The integer nearest to x (halves to even).
__device__ __forceinline__ float int_part(float x) { return __fadd_rn(__fadd_rn(x, 12582912.f), -12582912.f); }
// x's 11 leading bits (nearest): a whole number that fp16 holds, for a whole x below 2^15.
__device__ __forceinline__ float lead_part(float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xFFFFE000u); }
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 8 x 8 16-bit matrix, a row of two elements a lane, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// D = A(16x16 f16, row) . B(16x8 f16, col) + C.
__device__ __forceinline__ void mma_f16_c(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1,
                                          float c2, float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// The first unit of part i of n of a line of `total` units.
__device__ __forceinline__ int64_t cut(int64_t i, int64_t each, int64_t more) {
  return i * each + min(i, more);
}
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

// The SMs that tc_kernel leaves idle, or 0 if taking all SMs later is as fast:
// its tiles take about as long for 32 tokens as a unit here, its longest sequence
// thus as long as the wait for its SMs.  units: of a warp on all SMs.
__device__ __forceinline__ int idle_sms(const Args& a, float units) {
  const int lane = threadIdx.x & 31;
  int items = 0, longest = 0;
#pragma unroll 1
  for (int64_t b0 = 0; b0 < a.n_seqs; b0 += 32) {
    const Seq s = b0 + lane < a.n_seqs ? seq_of(a, b0 + lane) : Seq{};
    const int t = big_tiles(a, s.n);
    items += __reduce_add_sync(0xffffffffu, t);
    longest = max(longest, __reduce_max_sync(0xffffffffu, t ? s.len : 0));
  }
  const Waves waves(a, items * a.hkv);
  const int idle = waves.items == waves.whole ? 0 : a.sms - (waves.items - waves.whole) * waves.cut;
  longest /= waves.cut;
  return idle > 0 && units * (float)(a.sms - idle) * kUnit <= (float)longest * (float)idle ? idle : 0;
}

// Work: a segment is 4 NB query rows (tokens x heads of one KV head) of one
// sequence over all its tokens; its units are 32 tokens.  All units of all
// segments lie on one line that is cut evenly among the warps of a grid that
// fits the GPU at once, whatever the lengths are.  A warp's pieces of
// segments that other warps continue are joined in shared memory, and pieces
// that other CTAs continue go to the workspace for join_kernel.
//
// Each warp streams its tiles with bulk copies into its own two-stage ring.
//
// BESIDE: launched behind tc_kernel, which has waited for what came before when
// this kernel starts; the two run side by side on different SMs, and this grid
// ends (its first CTA does) after that one.
template <int D, int NG, int NB, bool BESIDE>
__global__ void __launch_bounds__(warps_of(D, NG, NB) * 32, ctas_per_sm(D, NG, NB)) attn_kernel(const Args a) {
  constexpr int NC = D / 32, NS = D / 64, G = D / NG, W = warps_of(D, NG, NB);
  constexpr int TB = tile_bytes(D, NG), PF = part_floats(D, NB), ROWS = rows_of(NB);
  constexpr uint32_t kEven = 0x000F000Fu, kOdd = 0x00F000F0u;  // codes, and 16 times them
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[W][kStages];
  __shared__ Line s_line;
  __shared__ SegInfo s_seg[W][2];           // kept pieces: at the warp's first unit, at its last
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  griddep_launch_dependents();
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[warp][i], 1);
    mbar_fence_init();
  }
  if constexpr (BESIDE) __syncwarp();
  else griddep_wait();

  // ---- the line of units, and where this warp begins on it
  auto tiles_of = [&](int n) { return n * a.r > a.big ? 0 : seq_tiles<ROWS>(n, a.r); };
  const int64_t cta = blockIdx.x;
  SegInfo* info = reinterpret_cast<SegInfo*>(a.ws);
  float* parts = reinterpret_cast<float*>(a.ws + (size_t)gridDim.x * sizeof(SegInfo));
  int64_t w_a, w_b, b, off;
  // Every warp sums all sequences for itself: no barrier, one latency for 256 of
  // them.  T is 32 bits wide unless the host's bound of the line is wider: all
  // warps of an SM do this at once, and the 64-bit sums and divisions took twice
  // the time (2.6 us of a 20 us call).  Loops stay rolled and there is one search:
  // unrolled copies made this 100 KB of code, and fetching instructions took most
  // of a short call's time.
  auto plan = [&](auto zero) -> bool {
    using T = decltype(zero);
    auto line_units = [&](int64_t b) -> T {
      if (b >= a.n_seqs) return 0;
      const Seq s = seq_of(a, b);
      return (T)seq_units(s.len) * (T)tiles_of(s.n) * (T)a.hkv;
    };
    const bool one = a.n_seqs == 1;
    auto scan = [&](T v) -> T {             // inclusive, over the lanes
      if (one) return __shfl_sync(0xffffffffu, v, 0);
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const T u = __shfl_up_sync(0xffffffffu, v, x);
        if (lane >= x) v += u;
      }
      return v;
    };
    auto div = [](T x, T y) -> T { return (T)((sizeof(T) == 4) ? (uint32_t)x / (uint32_t)y : quot(x, y)); };
    // A lane has up to eight neighbouring sequences at a time.
    const int per = a.n_seqs > 224 ? 8 : ((int)a.n_seqs + 31) / 32;
    auto some = [&](int64_t b0) -> T {
      T v = 0;
#pragma unroll 1
      for (int i = 0; i < per; ++i) v += line_units(b0 + lane * per + i);
      return v;
    };
    const T v_first = some(0), end_first = scan(v_first);
    T all = __shfl_sync(0xffffffffu, end_first, 31);
#pragma unroll 1
    for (int64_t b0 = 32 * per; b0 < a.n_seqs; b0 += 32 * per) all += __shfl_sync(0xffffffffu, scan(some(b0)), 31);
    T grid = (T)gridDim.x;
    if constexpr (BESIDE) {
      const int idle = idle_sms(a, (float)all / W / (float)gridDim.x);
      if (idle > 0) grid = (T)(gridDim.x / a.sms * idle);
    }
    const T n_ctas = max((T)1, min(grid, div(all + W - 1, W)));
    if (cta >= n_ctas || all == 0) return false;
    const T t_each = div(all, n_ctas), t_more = all - t_each * n_ctas, me = (T)cta;
    T first = me * t_each + min(me, t_more), last = first + t_each + (me < t_more ? 1 : 0), unit = first, o = 0;
    // Uncut, a CTA has the segments that begin in its part: steps 0 and 1 move its
    // ends to where segments begin.  Step 2 looks for this warp's first unit.
#pragma unroll 1
    for (int step = a.uncut ? 0 : 2; step < 3; ++step) {
      if (step == 2) {
        if (first >= last) return false;
        const T w_each = div(last - first, W), w_more = last - first - w_each * W, w = (T)warp;
        unit = first + w * w_each + min(w, w_more);
        w_a = unit;
        w_b = unit + w_each + (w < w_more ? 1 : 0);
      }
      // the sequence of the unit, and the unit within it
      b = 0;
      o = unit;
      if (!one && unit < all) {
        T base = 0, v = v_first, end = end_first;
        unsigned past;
#pragma unroll 1
        while (!(past = __ballot_sync(0xffffffffu, base + end > unit)) && b + 32 * per < a.n_seqs) {
          base += __shfl_sync(0xffffffffu, end, 31);
          b += 32 * per;
          v = some(b);
          end = scan(v);
        }
        const int who = past ? __ffs(past) - 1 : 0;
        o = unit - base - __shfl_sync(0xffffffffu, end - v, who);
        b += who * per;
        if (per > 1) {
          const T u = lane < per ? line_units(b + lane) : 0, sum = scan(u);
          const unsigned here = __ballot_sync(0xffffffffu, sum > o);
          const int at = here ? __ffs(here) - 1 : 0;
          b += at;
          o -= __shfl_sync(0xffffffffu, sum - u, at);
        }
      }
      if (step < 2) {
        if (unit < all) {
          const T nu = (T)seq_units(seq_of(a, b).len), rem = o - div(o, nu) * nu;
          if (rem) unit += nu - rem;
        }
        if (step == 0) {
          first = unit;
          unit = last;
        } else {
          last = unit;
        }
      }
    }
    off = o;
    if (tid == 0) s_line = {t_each, t_more, first, last, o, b, n_ctas};
    return true;
  };
  if (!(a.wide ? plan((int64_t)0) : plan((int32_t)0))) {
    if (tid == 0 && !a.uncut) info[cta].u0 = -1;
    if (BESIDE && cta == 0) griddep_wait();
    return;
  }
  if (lane < 2) s_seg[warp][lane].u0 = -1;
  uint8_t* ring = smem + (size_t)warp * kStages * 2 * TB;
  float* kept = reinterpret_cast<float*>(smem + (size_t)W * kStages * 2 * TB) + warp * PF;
  uint32_t phase = 0;                       // parity of each stage's next use
  for (int64_t at = w_a; at < w_b;) {
    const Seq s = seq_of(a, b);
    const int tiles = tiles_of(s.n), nu = seq_units(s.len);
    if (off >= (int64_t)nu * tiles * a.hkv) {  // the next sequence
      off = 0;
      ++b;
      continue;
    }
    const int64_t seg = quot(off, nu);
    const int u_first = (int)(off - seg * nu);
    const int u_count = (int)min((int64_t)(nu - u_first), w_b - at);
    const int kvh = tiles == 1 ? (int)seg : (int)quot(seg, tiles), tile = (int)(seg - (int64_t)kvh * tiles);

    // Rows of the tile: lane column g of B is row g / 2 (integer part, then
    // rest); scores, softmax and outputs of row c are with the lanes c.
    auto row_at = [&](int i, int& tok, int& hq) -> bool {
      const int rr = tile * ROWS + i;
      tok = s.n == 1 ? (rr >= a.r) : a.r == 1 ? rr : (int)((uint32_t)rr / (uint32_t)a.r);
      hq = kvh * a.r + rr - tok * a.r;
      return rr < s.n * a.r;
    };
    const int last_tok = s.n == 1 ? 0 : min(s.n - 1, (int)((uint32_t)(tile * ROWS + ROWS - 1) / (uint32_t)a.r));
    const int seg_len = max(0, min(s.len, s.len - s.n + last_tok + 1));  // no row sees further
    const int all_see = s.len - s.n + (s.n == 1 ? 0 : (int)((uint32_t)(tile * ROWS) / (uint32_t)a.r)) + 1;             // every row sees these
    const int u_live = min(u_first + u_count, (seg_len + kUnit - 1) / kUnit);

    // this lane's part of the query rows, on its way while the tiles are found
    float x[NB][NC][8];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      int tok, hq;
      const bool ok = row_at(nb * 4 + (g >> 1), tok, hq);
      const float* qr = a.q + ((s.row0 + tok) * a.h + hq) * D + 8 * c;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        float4 v0 = make_float4(0.f, 0.f, 0.f, 0.f), v1 = v0;
        if (ok) {
          v0 = *reinterpret_cast<const float4*>(qr + 32 * j);
          v1 = *reinterpret_cast<const float4*>(qr + 32 * j + 4);
        }
        x[nb][j][0] = v0.x; x[nb][j][1] = v0.y; x[nb][j][2] = v0.z; x[nb][j][3] = v0.w;
        x[nb][j][4] = v1.x; x[nb][j][5] = v1.y; x[nb][j][6] = v1.z; x[nb][j][7] = v1.w;
      }
    }

    // Tiles are fetched by the lanes that know where they are: lane i has the
    // place of tile 2 ids_at + i.
    const uint8_t* src = nullptr;
    uint32_t known = 0;                     // which of those are there
    int ids_at = -1024;
    auto issue = [&](int u, int stage) -> uint32_t {
      if (u - ids_at >= 16) {
        ids_at = u;
        const uint32_t tt = 2 * (uint32_t)u + lane, per = (uint32_t)a.bs / kTile;
        const bool in = tt < (uint32_t)(seg_len + kTile - 1) / kTile;
        const uint32_t page = in ? tt / per : 0;
        const int blk = in ? a.table[b * a.width + page] : -1;
        const bool ok = blk >= 0 && blk < a.n_blocks;
        if (in && !ok && a.err) atomicExch(a.err, 4);  // never read: its tokens are left out
        src = a.cache + (((int64_t)blk * a.hkv + kvh) * per + (tt - page * per)) * TB;
        known = __ballot_sync(0xffffffffu, ok);
      }
      const int at2 = 2 * (u - ids_at);
      const uint32_t has = known >> at2 & 3u;
      if (lane == 0) mbar_arrive_expect_tx(&full[warp][stage], __popc(has) * TB);
      __syncwarp();
      if ((lane >> 1) == u - ids_at && (has >> (lane & 1) & 1u))
        bulk_g2s(ring + (stage * 2 + (lane & 1)) * TB, src, TB, &full[warp][stage]);
      return has;
    };
    uint32_t there = 0;                     // which of a stage's tiles are there: two bits a stage
    for (int i = 0; i < kStages; ++i)
      if (u_first + i < u_live) there |= issue(u_first + i, i) << (2 * i);

    // ---- B operand of the scores: q * scale * log2(e) on an integer grid
    uint32_t qf[NB][NC][2][2];
    float qsum[NB][NG], qc[NB][NG][2], row_f[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float amax = 0.f, asum = 0.f;
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[nb][j][i] *= a.scale2;
          amax = fmaxf(amax, fabsf(x[nb][j][i]));
          asum += fabsf(x[nb][j][i]);
        }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      asum += __shfl_xor_sync(0xffffffffu, asum, 1);
      asum += __shfl_xor_sync(0xffffffffu, asum, 2);
      // the largest magnitude goes below 2^15, the sum of all below 2^20
      const int e = max(14, min(244, max(exp_field(amax), exp_field(asum) - 5)));
      const float up = pow2_field(268 - e);
      float sum[NG], grid[NG];              // of q, and of this column's fp16 values
#pragma unroll
      for (int n = 0; n < NG; ++n) sum[n] = grid[n] = 0.f;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum[j * 32 / G] += x[nb][j][i];
          const float v = x[nb][j][i] * up, hi = lead_part(rintf(v));
          y[i] = g & 1 ? v - hi : hi;
          if (i & 1) y[i] *= 0.0625f;       // odd nibbles count 16 times
        }
        // k = 2c, 2c + 1 and 2c + 8, 2c + 9: nibbles 0, 4 and 2, 6 (1, 5 and 3, 7)
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            qf[nb][j][p][i] = pack_f16x2(y[p + 2 * i], y[p + 2 * i + 4]);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qf[nb][j][p][i]));
            grid[j * 32 / G] += (f.x + f.y) * (p ? 16.f : 1.f);
          }
      }
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 1);
        sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 2);
        grid[n] += __shfl_xor_sync(0xffffffffu, grid[n], 1);
        grid[n] += __shfl_xor_sync(0xffffffffu, grid[n], 2);
        // from row g / 2 to row c: lanes 8c (integers) and 8c + 4 (rests)
        qsum[nb][n] = __shfl_sync(0xffffffffu, sum[n], 8 * c);
        qc[nb][n][0] = __shfl_sync(0xffffffffu, grid[n], 8 * c) * -0x1p-21f;
        qc[nb][n][1] = __shfl_sync(0xffffffffu, grid[n], 8 * c + 4) * -0x1p-21f;
      }
      row_f[nb] = __shfl_sync(0xffffffffu, pow2_field(e + 10), 8 * c);  // 2^24 / up
    }
    int limit[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      int tok, hq;
      const bool ok = row_at(nb * 4 + c, tok, hq);
      limit[nb] = ok ? max(0, min(s.len, s.len - s.n + tok + 1)) : 0;
    }

    // ---- online softmax over the units
    float m[NB], l[NB], mins[NB][NG];
    float o[NB][NS][2][2][2];               // [span][half][pair][nibble], times 2^-12
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb] = -INFINITY;
      l[nb] = 0.f;
#pragma unroll
      for (int n = 0; n < NG; ++n) mins[nb][n] = 0.f;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) o[nb][i][k >> 2][(k >> 1) & 1][k & 1] = 0.f;
    }
    // Row i of a tile's MMAs is token i ^ (i >> 1 & 1), so that the value rows
    // that the four lanes of a quad read together lie in different banks.
    const int tg = g ^ ((g >> 1) & 1);
    bool failed = false;
    for (int u = u_first, st = 0; u < u_live; ++u, st ^= 1) {
      if (!mbar_wait_t<0>(&full[warp][st], (phase >> st) & 1u)) {
        if (a.err) atomicExch(a.err, 6);
        failed = true;
        break;
      }
      phase ^= 1u << st;
      const uint8_t* buf = ring + st * 2 * TB;
      const uint32_t has = there >> (2 * st) & 3u;
      const bool whole_unit = has == 3u && (u + 1) * kUnit <= all_see;

      // scores of tokens tg and tg + 8 of both tiles
      float sc[NB][2][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        uint32_t wa[NC], wb[NC];
        lds<NC>(buf + t * TB + tg * (D / 2) + c * NC * 4, wa);
        lds<NC>(buf + t * TB + (tg + 8) * (D / 2) + c * NC * 4, wb);
        float acc[NB][NG][4];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          constexpr int kPer = G / 32;
          const uint32_t xa = wa[j] >> 8, xb = wb[j] >> 8;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float (&d)[4] = acc[nb][j / kPer];
            const float* z = qc[nb][j / kPer];
            if (j % kPer == 0)
              mma_f16_c(d, wa[j] & kEven, wb[j] & kEven, xa & kEven, xb & kEven, qf[nb][j][0][0],
                        qf[nb][j][0][1], z[0], z[1], z[0], z[1]);
            else
              mma_f16_16816(d, wa[j] & kEven, wb[j] & kEven, xa & kEven, xb & kEven,
                            qf[nb][j][0][0], qf[nb][j][0][1]);
            mma_f16_16816(d, wa[j] & kOdd, wb[j] & kOdd, xa & kOdd, xb & kOdd, qf[nb][j][1][0],
                          qf[nb][j][1][1]);
          }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) sc[nb][t][0] = sc[nb][t][1] = 0.f;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const float2* p = reinterpret_cast<const float2*>(buf + t * TB + k_params_at(D)) + n * kTile + tg;
          const float2 pa = p[0], pb = p[8];
          const float ma = fmaf(8.f, pa.x, pa.y), mb = fmaf(8.f, pb.x, pb.y);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const float (&d)[4] = acc[nb][n];
            sc[nb][t][0] = fmaf((d[0] + d[1]) * row_f[nb], pa.x, fmaf(qsum[nb][n], ma, sc[nb][t][0]));
            sc[nb][t][1] = fmaf((d[2] + d[3]) * row_f[nb], pb.x, fmaf(qsum[nb][n], mb, sc[nb][t][1]));
          }
        }
      }
      if (!whole_unit)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tt = u * kUnit + (i >> 1) * kTile + (i & 1) * 8 + tg;
            if (tt >= limit[nb] || !(has >> (i >> 1) & 1u)) sc[nb][i >> 1][i & 1] = -INFINITY;
          }
      float corr[NB];
      bool moved = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float mu = fmaxf(fmaxf(sc[nb][0][0], sc[nb][0][1]), fmaxf(sc[nb][1][0], sc[nb][1][1]));
        mu = fmaxf(mu, __shfl_xor_sync(0xffffffffu, mu, 4));
        mu = fmaxf(mu, __shfl_xor_sync(0xffffffffu, mu, 8));
        mu = fmaxf(mu, __shfl_xor_sync(0xffffffffu, mu, 16));
        const float m_new = fmaxf(m[nb], mu);
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        corr[nb] = ex2(m[nb] - ref);        // 0 while nothing was seen
        moved |= m_new != m[nb];
        m[nb] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& v = sc[nb][i >> 1][i & 1];
          const float p = ex2(v - ref);
          sum += p;
          v = v == -INFINITY ? -1.f : p;    // a negative p marks a masked token
        }
        l[nb] = fmaf(l[nb], corr[nb], sum);
      }
      if (__any_sync(0xffffffffu, moved))
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int n = 0; n < NG; ++n) mins[nb][n] *= corr[nb];
#pragma unroll
          for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) o[nb][i][k >> 2][(k >> 1) & 1][k & 1] *= corr[nb];
        }

      // Values, half a span (32 channels, one group) at a time: rows i of an
      // MMA are channel 4i + nibble, rows i + 8 the next one.  A unit's
      // products are summed apart and then added.
      uint32_t vw[2][4][NS];                // rows of this lane's 8 tokens
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = (i >> 1) * 8 + 2 * c + ((i & 1) ^ (c & 1));
          lds<NS>(buf + t * TB + v_codes_at(D) + row * (D / 2) + g * NS * 4, vw[t][i]);
        }
      uint32_t wf[NB][2][2];                // B operand: w of a group
      float base[NB][4], f_even[NB], f_odd[NB];
#pragma unroll
      for (int sp = 0; sp < NS; ++sp)
#pragma unroll
        for (int hv = 0; hv < 2; ++hv) {
          const int n = (64 * sp + 32 * hv) / G;
          if ((64 * sp + 32 * hv) % G == 0) {
            float2 vp[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              vp[i] = reinterpret_cast<const float2*>(buf + (i >> 1) * TB + v_params_at(D, NG))[n * kTile + (i & 1) * 8 + tg];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              float w[4], wmax = 0.f;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float p = sc[nb][i >> 1][i & 1];
                const bool in = !(p < 0.f);
                w[i] = in ? p * vp[i].x : 0.f;
                mins[nb][n] = in ? fmaf(p, fmaf(8.f, vp[i].x, vp[i].y), mins[nb][n]) : mins[nb][n];
                wmax = fmaxf(wmax, w[i]);
              }
              wmax = fmaxf(wmax, __shfl_xor_sync(0xffffffffu, wmax, 4));
              wmax = fmaxf(wmax, __shfl_xor_sync(0xffffffffu, wmax, 8));
              wmax = fmaxf(wmax, __shfl_xor_sync(0xffffffffu, wmax, 16));
              const int e = max(14, min(252, exp_field(wmax)));
              const float up = pow2_field(264 - e);
              f_even[nb] = pow2_field(e + 2);   // 2^24 / up, times 2^-12
              f_odd[nb] = f_even[nb] * 0.0625f;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float v = w[i] * up, hi = int_part(v);
                wf[nb][i >> 1][i & 1] = transpose8(pack_f16x2(hi, v - hi));
              }
              // -8 sum(w), for the rows of even and of odd nibbles
              const uint32_t z0 = 0x80088008u, z1 = 0x80808080u;  // -8, -128 times 2^-24
              mma_f16_c(base[nb], z0, z1, z0, z1, wf[nb][0][0], wf[nb][0][1], 0.f, 0.f, 0.f, 0.f);
              mma_f16_16816(base[nb], z0, z1, z0, z1, wf[nb][1][0], wf[nb][1][1]);
            }
          }
          uint32_t x[2][2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            x[t][0] = prmt(vw[t][0][sp], vw[t][1][sp], hv ? 0x7632 : 0x5410);
            x[t][1] = prmt(vw[t][2][sp], vw[t][3][sp], hv ? 0x7632 : 0x5410);
          }
#pragma unroll
          for (int pr = 0; pr < 2; ++pr) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              float d[4];
              mma_f16_c(d, x[0][0] & kEven, x[0][0] & kOdd, x[0][1] & kEven, x[0][1] & kOdd,
                        wf[nb][0][0], wf[nb][0][1], base[nb][0], base[nb][1], base[nb][2], base[nb][3]);
              mma_f16_16816(d, x[1][0] & kEven, x[1][0] & kOdd, x[1][1] & kEven, x[1][1] & kOdd,
                            wf[nb][1][0], wf[nb][1][1]);
              float (&oo)[2] = o[nb][sp][hv][pr];
              oo[0] = fmaf(d[0] + d[1], f_even[nb], oo[0]);
              oo[1] = fmaf(d[2] + d[3], f_odd[nb], oo[1]);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              x[t][0] >>= 8;
              x[t][1] >>= 8;
            }
          }
        }
      __syncwarp();                         // the stage's readers are done
      if (u + kStages < u_live)
        there = (there & ~(3u << (2 * st))) | issue(u + kStages, st) << (2 * st);
    }
    if (failed) {  // the copies still in flight, then out; the answer is not valid
      for (int st = 0; st < kStages; ++st) (void)mbar_wait_t<0>(&full[warp][st], (phase >> st) & 1u);
      break;
    }

    // ---- the piece's sums, in real units
    const bool whole = u_count == nu;
    const int64_t u0 = at - u_first;
    const int k = u0 <= w_a ? 0 : 1;
    // a piece at the warp's last unit lies in the ring, whose copies are all read
    float* piece = k ? reinterpret_cast<float*>(ring) : kept;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        l[nb] += __shfl_xor_sync(0xffffffffu, l[nb], x);
#pragma unroll
        for (int n = 0; n < NG; ++n) mins[nb][n] += __shfl_xor_sync(0xffffffffu, mins[nb][n], x);
      }
      int tok, hq;
      const bool ok = row_at(nb * 4 + c, tok, hq);
      float* dst = whole ? a.out + ((s.row0 + tok) * a.h + hq) * D : piece + (nb * 4 + c) * D;
      const float inv = !whole ? 1.f : l[nb] == 0.f ? 0.f : 1.f / l[nb];
      if (ok || !whole)
#pragma unroll
        for (int sp = 0; sp < NS; ++sp)
#pragma unroll
          for (int hv = 0; hv < 2; ++hv) {
            const float mn = mins[nb][(64 * sp + 32 * hv) / G];
            const float (&oo)[2][2] = o[nb][sp][hv];
            *reinterpret_cast<float4*>(dst + 64 * sp + 32 * hv + 4 * g) =
                make_float4(fmaf(oo[0][0], 4096.f, mn) * inv, fmaf(oo[0][1], 4096.f, mn) * inv,
                            fmaf(oo[1][0], 4096.f, mn) * inv, fmaf(oo[1][1], 4096.f, mn) * inv);
          }
      if (!whole && g == 0) {
        piece[ROWS * D + nb * 4 + c] = m[nb];
        piece[ROWS * D + ROWS + nb * 4 + c] = l[nb];
      }
    }
    if (!whole && lane == 0) {
      SegInfo& si = s_seg[warp][k];
      si.u0 = u0;
      si.u1 = u0 + nu;
      si.row0 = s.row0;
      si.n = s.n;
      si.kvh = kvh;
      si.tile = tile;
    }
    at += u_count;
    off += u_count;
  }

  // ---- for the join, and pieces of one segment in neighbouring warps, a row a warp
  if (tid == 0 && !a.uncut) {  // the segment cut by this CTA's beginning, joined in its name if that is its first cut
    const Seq s = seq_of(a, s_line.b);
    const int tiles = tiles_of(s.n), nu = seq_units(s.len);
    const Line l = s_line;
    const int64_t seg = quot(l.off, nu);
    SegInfo si;
    si.u0 = l.begin - (l.off - seg * nu);
    si.u1 = si.u0 + nu;
    si.row0 = s.row0;
    si.n = s.n;
    si.kvh = (int32_t)quot(seg, tiles);
    si.tile = (int32_t)(seg - (int64_t)si.kvh * tiles);
    const int64_t before = cut(cta - 1, l.each, l.more);
    int64_t last = cta;                     // the CTA that holds its last unit
    if (l.each > 0) last = max(cta, quot(si.u1 - 1, l.each + 1));
    while (last + 1 < l.ctas && cut(last + 1, l.each, l.more) < si.u1) ++last;
    si.parts = (int32_t)(last - (cta - 1) + 1);
    si.second = si.u0 > before;
    if (si.u0 == l.begin || si.u0 < before) si.u0 = -1;
    info[cta] = si;
  }
  __syncthreads();
  constexpr int V = D / 32;
  auto piece_at = [&](int i) -> const float* {
    return i & 1 ? reinterpret_cast<const float*>(smem + (size_t)(i >> 1) * kStages * 2 * TB)
                 : reinterpret_cast<const float*>(smem + (size_t)W * kStages * 2 * TB) + (i >> 1) * PF;
  };
  const int64_t begin = s_line.begin, end = s_line.end;
  // which of the 2 W places hold a piece and which begin another segment, a lane
  // each, and the tasks (rows of segments) up to there
  const int64_t my_u0 = lane < 2 * W ? s_seg[lane >> 1][lane & 1].u0 : -1;
  const unsigned used = __ballot_sync(0xffffffffu, my_u0 >= 0);
  const int prev = 31 - __clz(used & ((1u << lane) - 1u));
  const int64_t prev_u0 = __shfl_sync(0xffffffffu, my_u0, max(prev, 0));
  const bool is_first = my_u0 >= 0 && (prev < 0 || prev_u0 != my_u0);
  const unsigned first = __ballot_sync(0xffffffffu, is_first);
  int my_rows = 0;
  if (is_first) my_rows = min(ROWS, s_seg[lane >> 1][lane & 1].n * a.r - s_seg[lane >> 1][lane & 1].tile * ROWS);
  int tasks = my_rows;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, tasks, x);
    if (lane >= x) tasks += v;
  }
  const int all_tasks = __shfl_sync(0xffffffffu, tasks, 31);
#pragma unroll 1
  for (int task = warp; task < all_tasks; task += W) {
    const int i0 = __ffs(__ballot_sync(0xffffffffu, tasks > task)) - 1;
    const int row = task - __shfl_sync(0xffffffffu, tasks - my_rows, i0);
    const unsigned later = i0 == 31 ? 0u : first & ~((2u << i0) - 1u);
    const unsigned members = used & ~((1u << i0) - 1u) & (later ? (1u << (__ffs(later) - 1)) - 1u : ~0u);
    const SegInfo& si = s_seg[i0 >> 1][i0 & 1];
    const bool whole = si.u0 >= begin && si.u1 <= end;
    float* slot = parts + (size_t)(2 * cta + (si.u0 <= begin ? 0 : 1)) * PF;
    {
      // the members' maxima and sums, a lane each; then their outputs
      Merged<V> all;
      const bool in = members >> lane & 1u;
      const float* mine_p = piece_at(in ? lane : i0);
      const float pm = in ? mine_p[ROWS * D + row] : -INFINITY;
      float top = pm;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float f = ex2(pm - (top == -INFINITY ? 0.f : top));
      float pl = in ? mine_p[ROWS * D + ROWS + row] * f : 0.f;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) pl += __shfl_xor_sync(0xffffffffu, pl, x);
      all.m = top;
      all.l = pl;
#pragma unroll 1
      for (unsigned rest = members; rest; rest &= rest - 1) {
        const int who = __ffs(rest) - 1;
        float po[V];
        load_v<V>(piece_at(who) + row * D + lane * V, po);
        const float w = __shfl_sync(0xffffffffu, f, who);
#pragma unroll
        for (int x = 0; x < V; ++x) all.o[x] = fmaf(w, po[x], all.o[x]);
      }
      if (whole) {
        const int rr = si.tile * ROWS + row, tok = (int)((uint32_t)rr / (uint32_t)a.r);
        const int hq = si.kvh * a.r + rr - tok * a.r;
        store_v<V>(a.out + ((si.row0 + tok) * a.h + hq) * D + lane * V, all.o, all.l == 0.f ? 0.f : 1.f / all.l);
      } else {
        store_v<V>(slot + row * D + lane * V, all.o, 1.f);
        if (lane == 0) {
          slot[ROWS * D + row] = all.m;
          slot[ROWS * D + ROWS + row] = all.l;
        }
      }
    }
  }
  if (BESIDE && cta == 0) griddep_wait();
}

// Joins the segments that several CTAs share.  Block i: the segment that CTA
// i's beginning cuts, if that is the segment's first cut.  Its rows are shared
// by the warps, several warps a row where there are few; every result is taken
// in a fixed order, so it does not depend on timing.  Launch and latency, about
// 3 us, are its whole cost.  The blocks behind them
// join the parts of tc_kernel's items, four blocks an item and a warp a row.
constexpr int kJoinWarps = 16;
template <int D, int NB, bool BESIDE>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const Args a, int ctas, const float* tc_parts, int tc_tokens) {
  constexpr int PF = part_floats(D, NB), ROWS = rows_of(NB), V = D / 32;
  __shared__ __align__(16) float s_o[kJoinWarps][D];
  __shared__ float s_m[kJoinWarps], s_l[kJoinWarps];
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t cta = BESIDE && a.uncut ? blockIdx.x + ctas : blockIdx.x;
  if (BESIDE && cta >= ctas) {
    int b = 0, tile = 0, total = 0;
    find_tile(a, INT32_MAX, b, tile, total);
    const Waves waves(a, total * a.hkv);
    const int last = (int)(cta - ctas) / 4, item = waves.whole + last, kvh = item % a.hkv;  // of the last wave
    if (waves.cut == 1 || !find_tile(a, item / a.hkv, b, tile, total)) return;
    const Seq s = seq_of(a, b);
    const int splits = waves.parts(item, (tile_len(a, s, tile) + tc_tokens - 1) / tc_tokens);
    if (splits == 1) return;
    const int row0 = tile * kTcRows, rows = min(kTcRows, s.n * a.r - row0);
    for (int row = (int)(cta - ctas) % 4 * kJoinWarps + warp; row < rows; row += 4 * kJoinWarps) {
      Merged<V> all;
      for (int j = 0; j < splits; ++j) {
        const float* p = tc_parts + (size_t)(last * waves.cut + j) * tc_part_floats(D);
        float po[V];
        load_v<V>(p + row * D + lane * V, po);
        all.take(p[kTcRows * D + row], p[kTcRows * (D + 1) + row], po);
      }
      const int rr = row0 + row, tok = (int)((uint32_t)rr / (uint32_t)a.r), hq = kvh * a.r + rr - tok * a.r;
      store_v<V>(a.out + ((s.row0 + tok) * a.h + hq) * D + lane * V, all.o, all.l == 0.f ? 0.f : 1.f / all.l);
    }
    return;
  }
  const SegInfo si = reinterpret_cast<const SegInfo*>(a.ws)[cta];
  const float* parts = reinterpret_cast<const float*>(a.ws + (size_t)ctas * sizeof(SegInfo));
  if (si.u0 < 0) return;
  const int rows = min(ROWS, si.n * a.r - si.tile * ROWS);
  const int groups = rows == 1 ? kJoinWarps : rows == 2 ? kJoinWarps / 2 : kJoinWarps / (rows <= 4 ? 4 : rows <= 8 ? 8 : 16);
  const int row = warp / groups, grp = warp - row * groups;
  Merged<V> all;
  if (row < rows) {
    // the first part lies in CTA cta - 1, the others at the beginning of theirs
    auto part = [&](int j) { return parts + (size_t)(2 * (cta - 1 + j) + (j == 0 ? si.second : 0)) * PF; };
    for (int j0 = grp; j0 < si.parts; j0 += 4 * groups) {
      float pm[4], pl[4], po[4][V];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = j0 + i * groups;
        const float* p = part(min(j, si.parts - 1));
        pm[i] = j < si.parts ? p[ROWS * D + row] : -INFINITY;
        pl[i] = j < si.parts ? p[ROWS * D + ROWS + row] : 0.f;
        load_v<V>(p + row * D + lane * V, po[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j0 + i * groups < si.parts) all.take(pm[i], pl[i], po[i]);
    }
    store_v<V>(&s_o[warp][lane * V], all.o, 1.f);
    if (lane == 0) {
      s_m[warp] = all.m;
      s_l[warp] = all.l;
    }
  }
  __syncthreads();
  if (row >= rows || grp != 0) return;
  for (int i = 1; i < min(groups, si.parts); ++i) {
    float po[V];
    load_v<V>(&s_o[warp + i][lane * V], po);
    all.take(s_m[warp + i], s_l[warp + i], po);
  }
  const int rr = si.tile * ROWS + row, tok = (int)((uint32_t)rr / (uint32_t)a.r);
  const int hq = si.kvh * a.r + rr - tok * a.r;
  store_v<V>(a.out + ((si.row0 + tok) * a.h + hq) * D + lane * V, all.o, all.l == 0.f ? 0.f : 1.f / all.l);
}

int grid_of(int d, int ng, int nb) { return ctx()->num_sms * ctas_per_sm(d, ng, nb); }

size_t few_ws_bytes(int d) { return (ws_bytes(grid_of(d, 4, 1), d) + 255) / 256 * 256; }
size_t all_ws_bytes(int d) { return few_ws_bytes(d) + (tc_serves(d) ? tc_ws_bytes(d) : 0); }

template <int D, int NG, int NB, bool BESIDE>
int run_nb(const Args& a, cudaStream_t st) {
  const int smem = attn_smem(D, NG, NB);
  NIMF_TRY(allow_smem((const void*)attn_kernel<D, NG, NB, BESIDE>, smem));
  const int ctas = grid_of(D, NG, NB);
  NIMF_TRY(launch(attn_kernel<D, NG, NB, BESIDE>, dim3(ctas), warps_of(D, NG, NB) * 32, smem, st, 1, a));
  // items with parts are half a wave or less
  const int64_t tc_blocks = BESIDE ? 4 * std::min<int64_t>(tc_items(a), a.sms / 2) : 0;
  const int64_t blocks = (a.uncut ? 0 : ctas) + tc_blocks;
  if (blocks == 0) return NIMF_OK;
  return launch(join_kernel<D, NB, BESIDE>, dim3((unsigned)blocks), kJoinWarps * 32, 0, st, 1, a, ctas,
                (const float*)(a.ws + few_ws_bytes(D)), 128 / NG);
}

// 4 rows a segment where no sequence should have more of them for a KV head,
// 8 or 16 where one may: each pass over a sequence's tiles serves more rows,
// at more registers and partial results.  Beside sequences of many rows, which
// go elsewhere, the others are taken for decoding ones with one row a head.
template <int D, int NG, bool BESIDE>
int run_rows(const Args& a, int64_t rows, cudaStream_t st) {
  if (rows <= 4) return run_nb<D, NG, 1, BESIDE>(a, st);
  if constexpr (D <= 128)
    if (rows > 8) return run_nb<D, NG, 4, BESIDE>(a, st);
  return run_nb<D, NG, 2, BESIDE>(a, st);
}
template <int D, int NG>
int run_attn(const Args& a, int64_t max_new, cudaStream_t st) {
  if constexpr (D <= 128)
    if (a.big < INT32_MAX) return run_rows<D, NG, true>(a, a.r, st);
  return run_rows<D, NG, false>(a, max_new * a.r, st);
}

// Rows a KV head from which a sequence is worth the tensor-core kernel's tiles
// of 128.  With one group a head such a tile costs about what 16 rows cost here: 64
// ragged requests up to 4,096 tokens, 8 KV heads of 128, 20 rows of each a head
// take 121 us there and 132 here.  Finer groups shrink its tiles of tokens, which
// this rule leaves out: with groups of 64 the kernels meet at about 36 rows (20 rows
// 170 and 157 us), with groups of 32 at about 44 (312 and 225).
constexpr int kBigRows = 16;

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
  *bytes = (int64_t)kv4::all_ws_bytes(s.d);
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
      n_seqs < 0 || n_seqs > kv4::kMaxSeqs || max_blocks < 1 || max_blocks > INT32_MAX / s.bs || max_new < 0)
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
  if (workspace_bytes < (int64_t)kv4::all_ws_bytes(s.d))
    return set_error(NIMF_ERR_ARG, "kv4_attention: %lld bytes of workspace, nimf_kv4_attention_workspace asks for %lld",
                     (long long)workspace_bytes, (long long)kv4::all_ws_bytes(s.d));
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
  // Short contexts: a CTA takes whole segments, so nothing is left to join.  A
  // segment of 24 units costs a CTA two units more a warp (2 us) than a cut one,
  // the join's launch and latency 3 us.
  a.uncut = max_blocks * s.bs <= 24 * kv4::kUnit;
  // an upper bound of the line of units: every row tile over a whole table row
  a.wide = ((double)rows * a.r / 4 + (double)n_seqs) * s.hkv * ((double)max_blocks * s.bs / kv4::kUnit + 1) > 1e9;
  a.big = INT32_MAX;
  a.sms = ctx()->num_sms;
  if (kv4::tc_serves(s.d) && max_new * a.r > kv4::kBigRows) {
    a.big = kv4::kBigRows;
    NIMF_TRY(kv4::run_tc(a, s.d, s.d / s.group, a.ws + kv4::few_ws_bytes(s.d), st));
  }
  switch (s.d * 16 + s.d / s.group) {
    case 64 * 16 + 1: return kv4::run_attn<64, 1>(a, max_new, st);
    case 64 * 16 + 2: return kv4::run_attn<64, 2>(a, max_new, st);
    case 128 * 16 + 1: return kv4::run_attn<128, 1>(a, max_new, st);
    case 128 * 16 + 2: return kv4::run_attn<128, 2>(a, max_new, st);
    case 128 * 16 + 4: return kv4::run_attn<128, 4>(a, max_new, st);
    case 256 * 16 + 2: return kv4::run_attn<256, 2>(a, max_new, st);
    case 256 * 16 + 4: return kv4::run_attn<256, 4>(a, max_new, st);
    default: return kv4::run_attn<256, 8>(a, max_new, st);
  }
}

}  // extern "C"
