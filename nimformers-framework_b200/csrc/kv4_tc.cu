// kv4_tc.cu -- attention of many rows per sequence (prompts and chunks of
// them) over the 4-bit paged KV cache on tcgen05.
//
// One CTA holds 128 query rows (tokens x heads of one KV head) and walks over
// tiles of N = 128 / NG tokens (NG groups a head).  The formulas are those of
// kv4_attn.cu with codes centred at 8 and converted to fp16 once per tile:
//   S_g = [qh | ql] . (c - 8)^T            q in two fp16 terms, M = 128, N tokens
//   x_j = sum_g S_g s_gj + (m_gj + 8 s_gj) sum_g(q)
//   O_g += [wh | wl] . (c - 8),  w_j = p_j s_gj    in two fp16 terms from TMEM
// so each product runs twice, which is what float32's accuracy costs here; the
// floor is twice the plain flops at the tensor rate.  An output tile's sums
// run in TMEM over one tile of tokens only and are added to float32 registers
// between, so that the tensor core's cut-off additions stay few.
//
// Roles: two softmax warpgroups take turns at the tiles (even and odd ones),
// each with its own S and O columns, running maximum and sums, joined at the
// end, so the tensor core works on one tile while the other is in softmax; one
// warpgroup unpacks codes into the K and V operands (two buffers each); one
// warp issues the MMAs.  P overwrites S in place: 32 columns of scores become
// 16 columns of high and 16 of low terms.
#include <algorithm>

#include "kv4.cuh"
#include "tc_util.cuh"

namespace nimf {
namespace kv4 {

namespace {

constexpr int kTcRows = 128;
constexpr int kTcThreads = 512;     // 2 softmax warpgroups, unpack, MMA
constexpr int kUnpack0 = 256;       // first unpack thread
constexpr int kPrmSlots = 4;        // tiles whose scales and minima are held
constexpr int kFails = 6;           // error word of an expired wait

// Shared memory, byte offsets.
template <int D, int NG>
struct TcLayout {
  static constexpr int N = 128 / NG;
  static constexpr int Q = 0;                                   // [2 terms][128][D] fp16
  static constexpr int K = Q + 2 * kTcRows * D * 2;             // [2 buffers][N][D]
  static constexpr int V = K + 2 * N * D * 2;                   // [2 buffers][D][N]
  static constexpr int PRM = V + 2 * N * D * 2;                 // [slots][ks, km, vs, vm][128] float
  static constexpr int F = PRM + kPrmSlots * 4 * 128 * 4;       // [slots][NG] float
  static constexpr int RED = F + kPrmSlots * 4 * 4;             // [2][4] uint32
  static constexpr int BAR = RED + 32;                          // barriers
  static constexpr int SIZE = BAR + 256;
};

size_t part_bytes(int d) { return (size_t)kTcRows * (d + 2) * 4; }

// ------------------------------------------------------------ PTX
__device__ __forceinline__ void umma_f16_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}" ::"r"(
          tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
// 32 consecutive columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]),
        "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]),
        "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]),
        "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]),
        "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr));
}
// Two floats in one 64-bit register, and packed arithmetic on them.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pk(float lo, float hi) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float lo_of(f2 v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(f2 v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// Two half-word codes (even: bits 0..3, odd: bits 4..7) less 8 as fp16: the
// nibble masked into 1024 + c (1024 + 16 c), then one add (FMA).
__device__ __forceinline__ uint32_t code_even(uint32_t w) {
  uint32_t v = lop3_and_or(w, 0x000F000Fu, 0x64006400u), r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0xE408E408u));
  return r;
}
__device__ __forceinline__ uint32_t code_odd(uint32_t w) {
  uint32_t v = lop3_and_or(w, 0x00F000F0u, 0x64006400u), r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v), "r"(0x2C002C00u), "r"(0xD480D480u));
  return r;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Writes of this thread to shared memory, seen by the tensor core's proxy.
__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Tiles of 128 rows of a sequence here, and the sequence and tile of index i
// counted from the end (the last rows see most tokens: the longest go first).
__device__ __forceinline__ int big_tiles(const Args& a, int n) {
  return n * a.r > a.big ? (n * a.r + kTcRows - 1) / kTcRows : 0;
}
__device__ __forceinline__ bool find_tile(const Args& a, int index, int& b, int& tile) {
  const int lane = threadIdx.x & 31;
  int total = 0;
  for (int64_t b0 = 0; b0 < a.n_seqs; b0 += 32) {
    const int64_t x = b0 + lane;
    int t = x < a.n_seqs ? big_tiles(a, seq_of(a, x).n) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    total += t;
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

template <int D, int NG>
__global__ void __launch_bounds__(kTcThreads, 1)
    tc_kernel(const Args a, int splits, unsigned char* parts) {
  using L = TcLayout<D, NG>;
  constexpr int N = L::N, G = D / NG, NC = D / 32, NS = D / 64, TB = tile_bytes(D, NG);
  constexpr int SB_D = D * 16, SB_N = N * 16;   // 8-row groups of operands with D, N columns of K
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint32_t s_tmem;
  __shared__ int s_where[3];
  __shared__ int s_stop;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t *k_full = bar, *k_empty = bar + 2, *v_full = bar + 4, *v_empty = bar + 6;
  uint64_t *s_full = bar + 8, *p_full = bar + 10, *o_full = bar + 12, *prm_full = bar + 14;
  uint64_t *q_full = bar + 18, *all_done = bar + 19;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = blockIdx.x % splits, item = blockIdx.x / splits;
  const int kvh = item % a.hkv;

  griddep_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 128);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 128);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < kPrmSlots; ++i) mbar_init(&prm_full[i], 128);
    mbar_init(q_full, 256);
    mbar_init(all_done, 1);
    s_stop = 0;
    mbar_fence_init();
  }
  griddep_wait();
  if (warp == 0) {
    int b = 0, tile = 0;
    const bool ok = find_tile(a, item / a.hkv, b, tile);
    if (lane == 0) {
      s_where[0] = ok;
      s_where[1] = b;
      s_where[2] = tile;
    }
  }
  __syncthreads();
  if (!s_where[0]) return;                      // more CTAs than tiles: the host knows a bound
  const int b = s_where[1], tile = s_where[2];
  const Seq s = seq_of(a, b);
  const int rows = min(kTcRows, s.n * a.r - tile * kTcRows);
  const int first_tok = (int)((uint32_t)(tile * kTcRows) / (uint32_t)a.r);
  const int last_tok = (int)((uint32_t)(tile * kTcRows + rows - 1) / (uint32_t)a.r);
  const int seg_len = max(0, min(s.len, s.len - s.n + last_tok + 1));
  const int all_see = s.len - s.n + first_tok + 1;
  // this split's tiles of tokens
  const int nt_all = (seg_len + N - 1) / N;
  const int t_first = (int)((int64_t)nt_all * split / splits);
  const int nt = (int)((int64_t)nt_all * (split + 1) / splits) - t_first;

  if (warp == 0) {
    tmem_alloc(&s_tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  auto stopped = [&]() { return *reinterpret_cast<volatile int*>(&s_stop) != 0; };
  auto wait = [&](uint64_t* m, uint32_t parity) -> bool {
    for (uint32_t i = 0; i < kMaxSpin; ++i) {
      if (mbar_try_wait(m, parity)) return true;
      if (stopped()) return false;
    }
    *reinterpret_cast<volatile int*>(&s_stop) = 1;
    if (a.err) atomicExch(a.err, kFails);
    return false;
  };

  if (warp >= 12) {
    // ---------------------------------------------------------------- MMA issue
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 12) {
      const uint32_t id_s = idesc_n(N), id_o = idesc_n(G);
      const uint64_t dq = smem_desc(smem + L::Q, 128, SB_D);
      const uint64_t dk = smem_desc(smem + L::K, 128, SB_D);
      const uint64_t dv = smem_desc(smem + L::V, 128, SB_N);
      auto warp_wait = [&](uint64_t* m, uint32_t parity) -> bool {
        int ok = lane == 0 ? (int)wait(m, parity) : 0;
        return __shfl_sync(0xffffffffu, ok, 0) != 0;
      };
      // S_x = q . k of tile t (x = t & 1)
      auto scores = [&](int t) -> bool {
        const int x = t & 1;
        if (!warp_wait(&k_full[x], (t >> 1) & 1)) return false;
        tc_fence_after();
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int j = 0; j < G / 16; ++j)
              if (elect_one())
                umma_f16_ss(tmem + x * 128 + g * N,
                            dq + ((term * kTcRows * D * 2 + (g * G / 8 + 2 * j) * 128) >> 4),
                            dk + ((x * N * D * 2 + (g * G / 8 + 2 * j) * 128) >> 4), id_s,
                            term + j > 0 ? 1u : 0u);
        if (elect_one()) {
          umma_commit(&s_full[x]);
          umma_commit(&k_empty[x]);
        }
        __syncwarp();
        return true;
      };
      bool ok = warp_wait(q_full, 0);
      if (ok && nt > 0) ok = scores(0);
      if (ok && nt > 1) ok = scores(1);
      for (int t = 0; ok && t < nt; ++t) {
        const int x = t & 1, ph = (t >> 1) & 1;
        ok = warp_wait(&v_full[x], ph) && warp_wait(&p_full[x], ph);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int j = 0; j < N / 16; ++j)
#pragma unroll
            for (int term = 0; term < 2; ++term)
              if (elect_one())
                umma_f16_ts(tmem + 256 + x * D + g * G,
                            tmem + x * 128 + g * N + (j >> 1) * 32 + term * 16 + (j & 1) * 8,
                            dv + ((x * N * D * 2 + (g * G / 8) * SB_N + j * 256) >> 4), id_o,
                            term + j > 0 ? 1u : 0u);
        if (elect_one()) {
          umma_commit(&o_full[x]);
          umma_commit(&v_empty[x]);
        }
        __syncwarp();
        // the next scores of these columns wait until P there was used
        if (t + 2 < nt) ok = warp_wait(&o_full[x], ph) && scores(t + 2);
      }
      if (elect_one()) umma_commit(all_done);
      __syncwarp();
      (void)warp_wait(all_done, 0);             // nothing in flight when TMEM is given back
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- unpack
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int pt = tid - kUnpack0, pw = pt >> 5;
    const uint32_t per = (uint32_t)a.bs / kTile;
    // tile of 16 tokens at token position tok, or NULL
    auto place = [&](int tok, bool report) -> const uint8_t* {
      if (tok >= seg_len) return nullptr;
      const uint32_t tt = (uint32_t)tok / kTile, page = tt / per;
      const int blk = a.table[(int64_t)b * a.width + page];
      if (blk < 0 || blk >= a.n_blocks) {
        if (report && a.err) atomicExch(a.err, 4);
        return nullptr;
      }
      return a.cache + (((int64_t)blk * a.hkv + kvh) * per + (tt - page * per)) * TB;
    };
    constexpr int KI = N * D / 32 / 128;        // 16-byte pieces of K rows a thread
    constexpr int VI = (N * NS + 127) / 128;    // 8 x 8 blocks of V a thread
    float* prm = reinterpret_cast<float*>(smem + L::PRM);
    float* fac = reinterpret_cast<float*>(smem + L::F);
    volatile uint32_t* red = reinterpret_cast<volatile uint32_t*>(smem + L::RED);
    bool ok = true;                             // after an expired wait the rounds go on without waits
    uint4 kw[KI];
    float2 kp, vp;
    uint32_t vw[VI][8];
    // one tile's rows of K with all scales and minima, and its rows of V
    auto load_k = [&](int base) {
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int it = pt + i * 128, tok = it % N, part = it / N;
        const uint8_t* p = place(base + tok, part == 0);
        kw[i] = p ? *reinterpret_cast<const uint4*>(p + (tok % kTile) * (D / 2) + part * 16)
                  : make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
      }
      const int tok = pt % N, n = pt / N;
      const uint8_t* p = place(base + tok, false);
      kp = vp = make_float2(0.f, 0.f);
      if (p) {
        kp = *reinterpret_cast<const float2*>(p + k_params_at(D) + (n * kTile + tok % kTile) * 8);
        vp = *reinterpret_cast<const float2*>(p + v_params_at(D, NG) + (n * kTile + tok % kTile) * 8);
      }
    };
    auto load_v = [&](int base) {
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        const int it = pt + i * 128, g = it & 7, kb = (it >> 3) % (N / 8), sp = it / N;
        const uint8_t* p = it < N * NS ? place(base + kb * 8, false) : nullptr;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          vw[i][e] = p && base + kb * 8 + e < seg_len
                         ? *reinterpret_cast<const uint32_t*>(p + v_codes_at(D) + ((kb & 1) * 8 + e) * (D / 2) + (g * NS + sp) * 4)
                         : 0x88888888u;
      }
    };
    load_k(t_first * N);
    load_v(t_first * N);
    for (int t = 0; t < nt; ++t) {
      const int x = t & 1, slot = t % kPrmSlots, base = (t_first + t) * N;
      // The parameters' slot was last used four tiles ago; that tile's values
      // were found used up when V of the tile before last was written.
      // w = p s is brought to fp16's range by the largest s of the tile
      uint32_t big = vp.x > 0.f ? __float_as_uint(vp.x) : 0u;   // a NaN has no say
      big = __reduce_max_sync(0xffffffffu, big);
      if (lane == 0) red[x * 4 + pw] = big;
      named_barrier(1, 128);
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < N / 32; ++i) most = max(most, red[x * 4 + (pw * 32 / N) * (N / 32) + i]);
      const int e = max(20, min(254, (int)(most >> 23)));
      prm[slot * 512 + pt] = kp.x;
      prm[slot * 512 + 128 + pt] = fmaf(8.f, kp.x, kp.y);
      prm[slot * 512 + 256 + pt] = vp.x * pow2_field(268 - e);  // largest in [2^14, 2^15)
      prm[slot * 512 + 384 + pt] = fmaf(8.f, vp.x, vp.y);
      if (pt % N == 0) fac[slot * 4 + pt / N] = pow2_field(e - 14);
      mbar_arrive(&prm_full[slot]);
      // K: 8 channels of a token a 16-byte piece, in the order of Q's
      if (t >= 2) ok = ok && wait(&k_empty[x], ((t >> 1) - 1) & 1);
      uint8_t* kd = smem + L::K + x * N * D * 2;
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int it = pt + i * 128, tok = it % N, part = it / N;
        const uint32_t w4[4] = {kw[i].x, kw[i].y, kw[i].z, kw[i].w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int m = part * 4 + q, c = m / NC, j = m % NC;
          const uint32_t w = w4[q], w8 = w >> 8;
          *reinterpret_cast<uint4*>(kd + (tok >> 3) * SB_D + (j * 4 + c) * 128 + (tok & 7) * 16) =
              make_uint4(code_even(w), code_even(w8), code_odd(w), code_odd(w8));
        }
      }
      fence_async_shared();
      mbar_arrive(&k_full[x]);
      load_k(base + N);                         // on its way through the wait for V's buffer
      // V: 8 tokens of a channel a 16-byte piece; row n = 64 s + 8 i + g is
      // channel 64 s + 32 (i / 4) + 4 g + i % 4
      if (t >= 2) ok = ok && wait(&v_empty[x], ((t >> 1) - 1) & 1);
      uint8_t* vd = smem + L::V + x * N * D * 2;
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        const int it = pt + i * 128, g = it & 7, kb = (it >> 3) % (N / 8), sp = it / N;
        if (it < N * NS) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t xx[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) xx[p] = prmt(vw[i][2 * p], vw[i][2 * p + 1], h ? 0x7632 : 0x5410);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint4 o;
              o.x = k & 1 ? code_odd(xx[0] >> (k & 2) * 4) : code_even(xx[0] >> (k & 2) * 4);
              o.y = k & 1 ? code_odd(xx[1] >> (k & 2) * 4) : code_even(xx[1] >> (k & 2) * 4);
              o.z = k & 1 ? code_odd(xx[2] >> (k & 2) * 4) : code_even(xx[2] >> (k & 2) * 4);
              o.w = k & 1 ? code_odd(xx[3] >> (k & 2) * 4) : code_even(xx[3] >> (k & 2) * 4);
              *reinterpret_cast<uint4*>(vd + (sp * 8 + h * 4 + k) * SB_N + kb * 128 + g * 16) = o;
            }
          }
        }
      }
      fence_async_shared();
      mbar_arrive(&v_full[x]);
      load_v(base + N);
    }
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int wg = warp >> 2, row = tid & 127;  // both warpgroups hold the same rows
    const uint32_t lane_at = tmem + ((uint32_t)(warp & 3) << 21);
    const bool row_ok = row < rows;
    const int rr = tile * kTcRows + row;
    const int tok = (int)((uint32_t)rr / (uint32_t)a.r), hq = kvh * a.r + rr - tok * a.r;
    const int limit = row_ok ? max(0, min(s.len, s.len - s.n + tok + 1)) : 0;
    const int64_t at = ((s.row0 + tok) * a.h + hq) * D;
    float qs[NG], row_f;
    {
      // this row of q: the warpgroups write its high and its low terms
      const float4* q4 = reinterpret_cast<const float4*>(a.q + (row_ok ? at : 0));
      float amax = 0.f;
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float t = 0.f;
#pragma unroll 8
        for (int j = 0; j < G / 4; ++j) {
          const float4 v = row_ok ? q4[n * (G / 4) + j] : make_float4(0.f, 0.f, 0.f, 0.f);
          const float x0 = v.x * a.scale2, x1 = v.y * a.scale2, x2 = v.z * a.scale2, x3 = v.w * a.scale2;
          amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x0), fabsf(x1))), fmaxf(fabsf(x2), fabsf(x3)));
          t += (x0 + x1) + (x2 + x3);
        }
        qs[n] = t;
      }
      const int e = max(20, min(240, exp_field(amax)));
      const float up = pow2_field(268 - e);     // the largest magnitude in [2^14, 2^15)
      row_f = pow2_field(e - 14);
#pragma unroll
      for (int n = 0; n < NG; ++n) qs[n] *= up;
      uint8_t* qd = smem + L::Q + wg * kTcRows * D * 2 + (row >> 3) * SB_D + (row & 7) * 16;
#pragma unroll 4
      for (int j = 0; j < D / 8; ++j) {
        const float4 v0 = row_ok ? q4[2 * j] : make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 v1 = row_ok ? q4[2 * j + 1] : make_float4(0.f, 0.f, 0.f, 0.f);
        float y[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = y[i] * a.scale2 * up;
          const float h = __half2float(__float2half_rn(y[i]));
          y[i] = wg ? y[i] - h : h;
        }
        *reinterpret_cast<uint4*>(qd + j * 128) =
            make_uint4(pack_h2(y[0], y[4]), pack_h2(y[2], y[6]), pack_h2(y[1], y[5]), pack_h2(y[3], y[7]));
      }
      fence_async_shared();
      mbar_arrive(q_full);
    }
    float m = -INFINITY;
    f2 l2 = pk(0.f, 0.f), mins[NG], o[D / 2];
#pragma unroll
    for (int n = 0; n < NG; ++n) mins[n] = l2;
#pragma unroll
    for (int i = 0; i < D / 2; ++i) o[i] = l2;
    const f2 rf2 = pk(row_f, row_f);
    bool ok = true;
    for (int t = wg; ok && t < nt; t += 2) {
      const uint32_t ph = (uint32_t)(t >> 1) & 1u;
      const int slot = t % kPrmSlots, base = (t_first + t) * N;
      const float* prm = reinterpret_cast<const float*>(smem + L::PRM) + slot * 512;
      ok = wait(&prm_full[slot], (uint32_t)(t / kPrmSlots) & 1u) && wait(&s_full[wg], ph);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const bool cut = base + N > all_see;      // some row does not see all of the tile
      // x of chunk k's 32 tokens, out of the scores of every group
      auto scores = [&](f2 (&x)[16], int k) {
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          float sc[32];
          tmem_ld32(lane_at + wg * 128 + n * N + 32 * k, sc);
          tmem_wait_ld();
          const f2 q2 = pk(qs[n], qs[n]);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const ulonglong2 ks = *reinterpret_cast<const ulonglong2*>(prm + n * N + 32 * k + i);
            const ulonglong2 km = *reinterpret_cast<const ulonglong2*>(prm + 128 + n * N + 32 * k + i);
            x[i / 2] = fma2(pk(sc[i], sc[i + 1]), ks.x, n ? fma2(q2, km.x, x[i / 2]) : mul2(q2, km.x));
            x[i / 2 + 1] = fma2(pk(sc[i + 2], sc[i + 3]), ks.y, n ? fma2(q2, km.y, x[i / 2 + 1]) : mul2(q2, km.y));
          }
        }
        if (cut) {
          const int seen = limit - (base + 32 * k);  // this row sees so many of them
#pragma unroll
          for (int i = 0; i < 16; ++i)
            x[i] = pk(2 * i < seen ? lo_of(x[i]) : -INFINITY, 2 * i + 1 < seen ? hi_of(x[i]) : -INFINITY);
        }
      };
      // pass 1: the largest x
      float top = -INFINITY;
#pragma unroll 1
      for (int k = 0; k < N / 32; ++k) {
        f2 x[16];
        scores(x, k);
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaxf(lo_of(x[i]), hi_of(x[i])));
      }
      const float m_new = fmaxf(m, top * row_f);
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      const float corr = ex2(m - ref);          // 0 while nothing was seen
      m = m_new;
      const f2 corr2 = pk(corr, corr), neg = pk(-ref, -ref), minus = pk(-1.f, -1.f);
      l2 = mul2(l2, corr2);
#pragma unroll
      for (int n = 0; n < NG; ++n) mins[n] = mul2(mins[n], corr2);
      // pass 2: probabilities, and w's two terms in place of the scores.  The
      // loops over chunks stay loops: unrolled, the two warpgroups' code does
      // not fit the instruction cache and fetching it takes five times longer
      // than running it.
#pragma unroll 1
      for (int k = 0; k < N / 32; ++k) {
        f2 x[16];
        scores(x, k);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[i] = fma2(x[i], rf2, neg);
          x[i] = pk(ex2(lo_of(x[i])), ex2(hi_of(x[i])));
          l2 = add2(l2, x[i]);
        }
        const int seen = limit - (base + 32 * k);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const float* pv = prm + 256 + n * N + 32 * k;
          uint32_t w[32];                       // high terms, then low ones
          if (cut) {                            // 0 times a NaN that this row does not see is 0
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const f2 vm = *reinterpret_cast<const f2*>(pv + 128 + 2 * i), u = mul2(x[i], vm);
              mins[n] = add2(mins[n], pk(2 * i < seen ? lo_of(u) : 0.f, 2 * i + 1 < seen ? hi_of(u) : 0.f));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const ulonglong2 vm = *reinterpret_cast<const ulonglong2*>(pv + 128 + 2 * i);
              mins[n] = fma2(x[i], vm.x, mins[n]);
              mins[n] = fma2(x[i + 1], vm.y, mins[n]);
            }
          }
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const ulonglong2 vs = *reinterpret_cast<const ulonglong2*>(pv + 2 * i);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              f2 w2 = mul2(x[i + e], e ? vs.y : vs.x);
              if (cut) w2 = pk(2 * (i + e) < seen ? lo_of(w2) : 0.f, 2 * (i + e) + 1 < seen ? hi_of(w2) : 0.f);
              // the high term is w cut to 11 bits (exact in fp16), the low one the rest
              const float h0 = __uint_as_float((uint32_t)w2 & 0xFFFFE000u);
              const float h1 = __uint_as_float((uint32_t)(w2 >> 32) & 0xFFFFE000u);
              const f2 rest = fma2(pk(h0, h1), minus, w2);
              w[i + e] = pack_h2(h0, h1);
              w[16 + i + e] = pack_h2(lo_of(rest), hi_of(rest));
            }
          }
          tmem_st32(lane_at + wg * 128 + n * N + 32 * k, w);
        }
      }
      // what the slot holds is in registers before the unpack warps may fill it again
      f2 f[NG];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const float v = reinterpret_cast<const float*>(smem + L::F)[slot * 4 + n];
        f[n] = pk(v, v);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[wg]);
      if (__any_sync(0xffffffffu, corr != 1.f))
#pragma unroll
        for (int i = 0; i < D / 2; ++i) o[i] = mul2(o[i], corr2);
      // the tile's sums of values
      ok = __all_sync(0xffffffffu, wait(&o_full[wg], ph));
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        float acc[32];
        tmem_ld32(lane_at + 256 + wg * D + 32 * k, acc);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[16 * k + i] = fma2(pk(acc[2 * i], acc[2 * i + 1]), f[32 * k / G], o[16 * k + i]);
      }
      tc_fence_before();
    }
    // ---- the two warpgroups' results; the operands' memory is free
    named_barrier(2, 256);
    float l = lo_of(l2) + hi_of(l2);
    float* xo = reinterpret_cast<float*>(smem + L::Q);      // [D][128]
    float* xs = reinterpret_cast<float*>(smem + L::PRM);    // m, l, minima [128]
    if (wg == 1) {
#pragma unroll
      for (int i = 0; i < D / 2; ++i) {
        xo[(2 * i) * 128 + row] = lo_of(o[i]);
        xo[(2 * i + 1) * 128 + row] = hi_of(o[i]);
      }
      xs[row] = m;
      xs[128 + row] = l;
#pragma unroll
      for (int n = 0; n < NG; ++n) xs[(2 + n) * 128 + row] = lo_of(mins[n]) + hi_of(mins[n]);
    }
    named_barrier(2, 256);
    if (wg == 0 && row_ok) {
      const float m1 = xs[row], top = fmaxf(m, m1), ref = top == -INFINITY ? 0.f : top;
      const float f0 = ex2(m - ref), f1 = ex2(m1 - ref);
      l = l * f0 + xs[128 + row] * f1;
      const bool whole = splits == 1;
      float* part = reinterpret_cast<float*>(parts + (size_t)blockIdx.x * kTcRows * (D + 2) * 4);
      float* dst = whole ? a.out + at : part + row * D;
      const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int sp = 0; sp < NS; ++sp)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = (64 * sp + 32 * h) / G;
          const float mn = (lo_of(mins[n]) + hi_of(mins[n])) * f0 + xs[(2 + n) * 128 + row] * f1;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int c = 64 * sp + 8 * (4 * h + i) + g;
              const float mine = c & 1 ? hi_of(o[c / 2]) : lo_of(o[c / 2]);
              v[i] = (mine * f0 + xo[c * 128 + row] * f1 + mn) * inv;
            }
            *reinterpret_cast<float4*>(dst + 64 * sp + 32 * h + 4 * g) = make_float4(v[0], v[1], v[2], v[3]);
          }
        }
      if (!whole) {
        part[kTcRows * D + row] = top;
        part[kTcRows * (D + 1) + row] = l;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, kTmemCols);
}

// Joins the splits of each tile of rows, in their order; a warp a row.
template <int D>
__global__ void __launch_bounds__(512) tc_join_kernel(const Args a, int splits, const unsigned char* parts) {
  constexpr int V = D / 32;
  __shared__ int s_where[3];
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int item = blockIdx.x, kvh = item % a.hkv;
  if (warp == 0) {
    int b = 0, tile = 0;
    const bool ok = find_tile(a, item / a.hkv, b, tile);
    if (lane == 0) {
      s_where[0] = ok;
      s_where[1] = b;
      s_where[2] = tile;
    }
  }
  __syncthreads();
  if (!s_where[0]) return;
  const Seq s = seq_of(a, s_where[1]);
  const int row0 = s_where[2] * kTcRows, rows = min(kTcRows, s.n * a.r - row0);
  for (int row = blockIdx.y * 16 + warp; row < rows; row += gridDim.y * 16) {
    Merged<V> all;
    for (int j = 0; j < splits; ++j) {
      const float* p = reinterpret_cast<const float*>(parts + (size_t)(item * splits + j) * kTcRows * (D + 2) * 4);
      float po[V];
      load_v<V>(p + row * D + lane * V, po);
      all.take(p[kTcRows * D + row], p[kTcRows * (D + 1) + row], po);
    }
    const int rr = row0 + row, tok = (int)((uint32_t)rr / (uint32_t)a.r), hq = kvh * a.r + rr - tok * a.r;
    store_v<V>(a.out + ((s.row0 + tok) * a.h + hq) * D + lane * V, all.o, all.l == 0.f ? 0.f : 1.f / all.l);
  }
}

int sms() {
  Context* c = ctx();
  return c ? c->num_sms : 148;
}

template <int D, int NG>
int run(const Args& a, int64_t max_blocks, unsigned char* ws, cudaStream_t st) {
  using L = TcLayout<D, NG>;
  const int64_t rows = a.rows * a.r;
  const int64_t tiles = rows / kTcRows + std::min<int64_t>(a.n_seqs, rows / (a.big + 1));
  const int64_t items = tiles * a.hkv;
  if (items == 0) return NIMF_OK;
  // With fewer tiles of rows than SMs the tokens are split too, down to four
  // tiles of them a CTA.
  const int64_t deep = std::max<int64_t>(1, max_blocks * a.bs / (4 * L::N));
  const int splits = items >= sms() ? 1 : (int)std::min<int64_t>(deep, 2 * sms() / items);
  NIMF_TRY(allow_smem((const void*)tc_kernel<D, NG>, L::SIZE));
  NIMF_TRY(launch(tc_kernel<D, NG>, dim3((unsigned)(items * splits)), kTcThreads, L::SIZE, st, 1, a, splits, ws));
  if (splits == 1) return NIMF_OK;
  return launch(tc_join_kernel<D>, dim3((unsigned)items, 4), 512, 0, st, 1, a, splits, (const unsigned char*)ws);
}

}  // namespace

bool tc_serves(int d) { return d <= 128; }
size_t tc_ws_bytes(int d) { return 2 * (size_t)sms() * part_bytes(d); }

int run_tc(const Args& a, int d, int ng, int64_t max_blocks, unsigned char* ws, cudaStream_t st) {
  switch (d * 16 + ng) {
    case 64 * 16 + 1: return run<64, 1>(a, max_blocks, ws, st);
    case 64 * 16 + 2: return run<64, 2>(a, max_blocks, ws, st);
    case 128 * 16 + 1: return run<128, 1>(a, max_blocks, ws, st);
    case 128 * 16 + 2: return run<128, 2>(a, max_blocks, ws, st);
    default: return run<128, 4>(a, max_blocks, ws, st);
  }
}

}  // namespace kv4
}  // namespace nimf
