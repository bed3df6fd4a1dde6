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
// floor is twice the plain flops at the tensor rate.  The tensor core cuts what
// an addition shifts out, always towards zero: so the low terms are summed first,
// while the sum is small, and an output tile's sums run in TMEM over one tile of
// tokens only and are added to float32 registers between.
//
// Roles: eight softmax warps of 16 rows; four warps that unpack codes into the K
// and V operands (two buffers each); one warp that issues the MMAs.  S and O have
// two buffers too: while tile t is in softmax the tensor core multiplies the
// values of tile t - 1 and the keys of tile t + 1.  P overwrites S in place: 16
// columns of scores become 8 of high and 8 of low terms.
// Softmax reads TMEM in the MMA fragment shape (a lane 2 rows x every fourth pair
// of columns): scales and minima are per column, and a lane with whole rows loads
// four times as many of them, which alone took longer than the products.
//
// Bounded by that chain of a softmax warp, 3 us a tile of 128 tokens; the tensor
// cores are 39 % busy: 2,048 rows of 6,144 tokens with 32 heads of 128 take 429 us
// (400 TFLOP/s with every product counted once), with groups of 64 706 us, of 32
// 1,353 us (captured calls over two sets of buffers).
#include <algorithm>
#include <type_traits>

#include "kv4.cuh"
#include "tc_util.cuh"

namespace nimf {
namespace kv4 {

namespace {

constexpr int kTcThreads = 512;     // 8 softmax warps, 4 of unpack, 1 of MMA issue
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
  static constexpr int PRM = V + 2 * N * D * 2;                 // [slots][K, V][64] {s, s, m, m}
  static constexpr int F = PRM + kPrmSlots * 4 * 128 * 4;       // [slots][NG] float
  static constexpr int RED = F + kPrmSlots * 4 * 4;             // [2][4] uint32
  static constexpr int ROW = RED + 32;                          // [1 + NG][128]: row_f, sums of q
  static constexpr int BAR = ROW + (1 + NG) * 128 * 4;                 // barriers
  static constexpr int SIZE = BAR + 256;
};

// ------------------------------------------------------------ PTX
// Descriptors (smem_desc's) as their two halves: the upper one is a constant of
// the operand, the lower one an address that offsets are added to.
__host__ __device__ constexpr uint32_t desc_hi(uint32_t sbo) { return ((sbo >> 4) & 0x3FFFu) | 1u << 14; }
__device__ __forceinline__ uint32_t desc_lo(const void* p, uint32_t lbo) {
  return ((smem_addr(p) >> 4) & 0x3FFFu) | ((lbo >> 4) & 0x3FFFu) << 16;
}
__device__ __forceinline__ void mma_ss(uint32_t tmem_d, uint32_t a, uint32_t a_hi, uint32_t b,
                                       uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n mov.b64 da, {%1, %2};\n mov.b64 db, {%3, %4};\n"
      " setp.ne.b32 p, %6, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, {%7, %7, %7, %7}, p;\n}" ::"r"(tmem_d),
      "r"(a), "r"(a_hi), "r"(b), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b, uint32_t b_hi,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n mov.b64 db, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, {%6, %6, %6, %6}, p;\n}" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
// 16 TMEM lanes x 8 columns a group: lane t holds columns 2 (t % 4), + 1 of row
// t / 4 (registers 0, 1) and of row t / 4 + 8 (2, 3).
__device__ __forceinline__ void tmem_ld_frag(uint32_t at, float (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
      : "r"(at));
}
__device__ __forceinline__ void tmem_ld_frag(uint32_t at, float (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(at));
}
// 16 TMEM lanes x 4 columns a group: lane t holds column t % 4 of rows t / 4 and
// t / 4 + 8.
__device__ __forceinline__ void tmem_st_frag(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_frag(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
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

template <int D, int NG>
__global__ void __launch_bounds__(kTcThreads, 1)
    tc_kernel(const Args a, unsigned char* parts) {
  using L = TcLayout<D, NG>;
  constexpr int N = L::N, G = D / NG, NC = D / 32, NS = D / 64, TB = tile_bytes(D, NG);
  constexpr int SB_D = D * 16, SB_N = N * 16;   // 8-row groups of operands with D, N columns of K
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint32_t s_tmem;
  __shared__ int s_where[4];
  __shared__ int s_stop, s_missing;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t *k_full = bar, *k_empty = bar + 2, *v_full = bar + 4, *v_empty = bar + 6;
  uint64_t *s_full = bar + 8, *p_full = bar + 10, *o_full = bar + 12, *prm_full = bar + 14;
  uint64_t *q_full = bar + 18, *all_done = bar + 19;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 128);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 128);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 256);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < kPrmSlots; ++i) mbar_init(&prm_full[i], 128);
    mbar_init(q_full, 256);
    mbar_init(all_done, 1);
    s_stop = s_missing = 0;
    mbar_fence_init();
  }
  // In this order, and before any CTA returns: attn_kernel<.., BESIDE = true> starts
  // when all CTAs are past here, and takes what came before this kernel for complete.
  griddep_wait();
  griddep_launch_dependents();
  if (warp == 0) {
    // the items' number gives their parts, so the item of a CTA is known after it
    int b = 0, tile = 0, total = 0;
    find_tile(a, INT32_MAX, b, tile, total);
    const Waves wv(a, total * a.hkv);
    const int over = (int)blockIdx.x - wv.whole, item = over < 0 ? blockIdx.x : wv.whole + over / wv.cut;
    const bool ok = find_tile(a, item / a.hkv, b, tile, total);
    if (lane == 0) {
      s_where[0] = ok;
      s_where[1] = b;
      s_where[2] = tile;
      s_where[3] = wv.items;
    }
  }
  __syncthreads();
  if (!s_where[0]) return;                      // more CTAs than tiles: the host knows a bound
  const Waves waves(a, s_where[3]);
  const int over = (int)blockIdx.x - waves.whole;
  const int item = over < 0 ? blockIdx.x : waves.whole + over / waves.cut, split = over < 0 ? 0 : over % waves.cut;
  const int kvh = item % a.hkv;
  const int b = s_where[1], tile = s_where[2];
  const Seq s = seq_of(a, b);
  const int rows = min(kTcRows, s.n * a.r - tile * kTcRows);
  const int first_tok = (int)((uint32_t)(tile * kTcRows) / (uint32_t)a.r);
  const int seg_len = tile_len(a, s, tile);
  const int all_see = s.len - s.n + first_tok + 1;
  // this split's tiles of tokens
  const int nt_all = (seg_len + N - 1) / N;
  const int splits = waves.parts(item, nt_all);
  if (split >= splits) return;
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

  // The unpack warps are ahead: their polls leave the issue slots to softmax.
  auto slow_wait = [&](uint64_t* m, uint32_t parity) -> bool {
    for (uint32_t i = 0; i < kMaxSpin; ++i) {
      if (mbar_try_wait_sleep(m, parity, 100u)) return true;
      if (stopped()) return false;
    }
    return wait(m, parity);
  };

  if (warp >= 12) {
    // ---------------------------------------------------------------- MMA issue
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 12) {
      // Everything an MMA is given is a constant away from warp-uniform values
      // (the buffer is a template argument, TMEM's base went through a warp
      // reduction): operands in per-thread registers cost six moves to uniform
      // ones an MMA, and the issue then takes twice the MMAs' own time.
      const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
      const uint32_t id_s = idesc_n(N), id_o = idesc_n(G);
      const uint32_t dq0 = desc_lo(smem + L::Q, 128), dk0 = desc_lo(smem + L::K, 128), dv0 = desc_lo(smem + L::V, 128);
      auto warp_wait = [&](uint64_t* m, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, wait(m, parity)) != 0;
      };
      // S = q . k of tile t in buffer x = t & 1
      auto scores = [&](auto buffer, int t) -> bool {
        constexpr int x = decltype(buffer)::value;
        if (!warp_wait(&k_full[x], (t >> 1) & 1)) return false;
        tc_fence_after();
        uint32_t td = tm, dq = dq0, dk = dk0;   // opaque: not to be hoisted as 32 sums and spilled
        asm volatile("" : "+r"(td), "+r"(dq), "+r"(dk));
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int term = 1; term >= 0; --term)
#pragma unroll
            for (int j = 0; j < G / 16; ++j)
              if (elect_one())
                mma_ss(td + (x * 128 + g * N), dq + ((term * kTcRows * D * 2 + (g * G / 8 + 2 * j) * 128) >> 4),
                       desc_hi(SB_D), dk + ((x * N * D * 2 + (g * G / 8 + 2 * j) * 128) >> 4), desc_hi(SB_D),
                       id_s, term == 0 || j > 0 ? 1u : 0u);
        if (elect_one()) {
          umma_commit(&s_full[x]);
          umma_commit(&k_empty[x]);
        }
        __syncwarp();
        return true;
      };
      auto values = [&](auto buffer, int t) -> bool {
        constexpr int x = decltype(buffer)::value;
        const uint32_t ph = (t >> 1) & 1;
        if (!warp_wait(&v_full[x], ph) || !warp_wait(&p_full[x], ph)) return false;
        tc_fence_after();
        uint32_t td = tm, dv = dv0;
        asm volatile("" : "+r"(td), "+r"(dv));
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int term = 1; term >= 0; --term)
#pragma unroll
            for (int j = 0; j < N / 16; ++j)
              if (elect_one())
                mma_ts(td + (256 + x * D + g * G), td + (x * 128 + g * N + j * 16 + term * 8),
                       dv + ((x * N * D * 2 + (g * G / 8) * SB_N + j * 256) >> 4), desc_hi(SB_N), id_o,
                       term == 0 || j > 0 ? 1u : 0u);
        if (elect_one()) {
          umma_commit(&o_full[x]);
          umma_commit(&v_empty[x]);
        }
        __syncwarp();
        // the next scores of these columns wait until P there was used
        return t + 2 >= nt || (warp_wait(&o_full[x], ph) && scores(buffer, t + 2));
      };
      const std::integral_constant<int, 0> even{};
      const std::integral_constant<int, 1> odd{};
      bool ok = warp_wait(q_full, 0);
      if (ok && nt > 0) ok = scores(even, 0);
      if (ok && nt > 1) ok = scores(odd, 1);
      for (int t = 0; ok && t < nt; t += 2) {
        ok = values(even, t);
        if (ok && t + 1 < nt) ok = values(odd, t + 1);
      }
      if (elect_one()) umma_commit(all_done);
      __syncwarp();
      // nothing is in flight when TMEM is given back, after an expired wait neither
      for (uint32_t i = 0; i < kMaxSpin && !mbar_try_wait(all_done, 0); ++i) {}
      __syncwarp();
    } else {
      // The three warps with nothing else to do look for blocks outside the cache,
      // beside the loads of q, so that softmax asks which tokens are missing only where
      // some are: asking in every tile took 1.5 % of a long prompt's time, this 0.4 %
      // (1.4 % of a step whose row tiles have an SM each; 4 % with four entries of a
      // lane in flight: more code, fetched cold).
      const int32_t* row_of_table = a.table + (int64_t)b * a.width;
      const uint32_t end = (uint32_t)min(seg_len, (t_first + nt) * N), per = (uint32_t)a.bs;
      bool missing = false;
      for (uint32_t page = (uint32_t)(t_first * N) / per + (tid - 13 * 32); page * per < end; page += 2 * 96) {
        int blk[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) blk[i] = (page + i * 96) * per < end ? row_of_table[page + i * 96] : 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) missing |= (uint32_t)blk[i] >= (uint32_t)a.n_blocks;
      }
      if (missing) s_missing = 1;
      __syncwarp();
      asm volatile("bar.arrive 2, %0;" ::"n"(256 + 96) : "memory");
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- unpack
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int pt = tid - kUnpack0, pw = pt >> 5;
    const uint32_t per = (uint32_t)a.bs / kTile;
    // The place of a token that moves on by N a tile: its block-table entry and
    // its tile within the block, kept without divisions.
    // The entry is loaded a tile ahead: it has to be there to load the codes.
    struct Walk {
      int tok, blk;
      uint32_t page, rem;
    };
    const int32_t* row_of_table = a.table + (int64_t)b * a.width;
    auto walk_at = [&](int tok) -> Walk {
      const uint32_t tt = (uint32_t)tok / kTile, page = tt / per;
      return Walk{tok, tok < seg_len ? row_of_table[page] : -1, page, tt - page * per};
    };
    auto step = [&](Walk& w, bool report) -> const uint8_t* {
      const uint8_t* p = nullptr;
      if (w.tok < seg_len) {
        const int blk = w.blk;
        if (blk >= 0 && blk < a.n_blocks)
          p = a.cache + (((int64_t)blk * a.hkv + kvh) * per + w.rem) * TB;
        else if (report && a.err)
          atomicExch(a.err, 4);                 // never read: softmax leaves its tokens out
      }
      w.tok += N;
      w.rem += N / kTile;
      while (w.rem >= per) {
        w.rem -= per;
        ++w.page;
      }
      w.blk = w.tok < seg_len ? row_of_table[w.page] : -1;
      return p;
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
    // K: token pt % N, every NG-th 16-byte piece of its row from pt / N on, and
    // the scales and minima of its group pt / N.  V: 8 tokens from 8 kb on, the
    // words of lane group g of one span or both.
    const int k_tok = pt % N, k_part = pt / N, vg = pt & 7, v_kb = (pt >> 3) % (N / 8), v_sp = pt / N;
    Walk wk = walk_at(t_first * N + k_tok), wv = walk_at(t_first * N + v_kb * 8);
    auto load_k = [&]() {
      const uint8_t* p = step(wk, k_part == 0);
      kp = vp = make_float2(-0.f, 0.f);         // a scale of -0 stands for a token that is not there
#pragma unroll
      for (int i = 0; i < KI; ++i) kw[i] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
      if (p) {
        const uint4* row = reinterpret_cast<const uint4*>(p + (k_tok % kTile) * (D / 2)) + k_part;
#pragma unroll
        for (int i = 0; i < KI; ++i) kw[i] = row[i * NG];
        kp = *reinterpret_cast<const float2*>(p + k_params_at(D) + (k_part * kTile + k_tok % kTile) * 8);
        vp = *reinterpret_cast<const float2*>(p + v_params_at(D, NG) + (k_part * kTile + k_tok % kTile) * 8);
      }
    };
    auto load_v = [&]() {
      const int left = seg_len - wv.tok;        // of these 8 tokens
      const uint8_t* p = step(wv, false);
      if (VI * 128 > N * NS && pt >= N * NS) p = nullptr;
#pragma unroll
      for (int i = 0; i < VI; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          vw[i][e] = 0x88888888u;
          if (p && e < left)
            vw[i][e] = *reinterpret_cast<const uint32_t*>(p + v_codes_at(D) + ((v_kb & 1) * 8 + e) * (D / 2) +
                                                          (vg * NS + v_sp + i) * 4);
        }
    };
    load_k();
    load_v();
    for (int t = 0; t < nt; ++t) {
      const int x = t & 1, slot = t % kPrmSlots;
      // K: 8 channels of a token a 16-byte piece, in the order of Q's
      if (t >= 2) ok = ok && slow_wait(&k_empty[x], ((t >> 1) - 1) & 1);
      uint8_t* kd = smem + L::K + x * N * D * 2;
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int part = k_part + i * NG;
        const uint32_t w4[4] = {kw[i].x, kw[i].y, kw[i].z, kw[i].w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int m = part * 4 + q, c = m / NC, j = m % NC;
          const uint32_t w = w4[q], w8 = w >> 8;
          *reinterpret_cast<uint4*>(kd + (k_tok >> 3) * SB_D + (j * 4 + c) * 128 + (k_tok & 7) * 16) =
              make_uint4(code_even(w), code_even(w8), code_odd(w), code_odd(w8));
        }
      }
      fence_async_shared();
      mbar_arrive(&k_full[x]);
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
      float* pp = prm + slot * 512 + (pt >> 1) * 4 + (pt & 1);
      pp[0] = kp.x;
      pp[2] = fmaf(8.f, kp.x, kp.y);
      pp[256] = vp.x * pow2_field(268 - e);     // largest in [2^14, 2^15)
      pp[258] = fmaf(8.f, vp.x, vp.y);
      if (pt % N == 0) fac[slot * 4 + pt / N] = pow2_field(e - 14);
      mbar_arrive(&prm_full[slot]);
      load_k();                       // on its way through the wait for V's buffer
      // V: 8 tokens of a channel a 16-byte piece; row n = 64 s + 8 i + g is
      // channel 64 s + 32 (i / 4) + 4 g + i % 4
      if (t >= 2) ok = ok && slow_wait(&v_empty[x], ((t >> 1) - 1) & 1);
      uint8_t* vd = smem + L::V + x * N * D * 2;
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        if (VI * 128 <= N * NS || pt < N * NS) {
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
              *reinterpret_cast<uint4*>(vd + ((v_sp + i) * 8 + h * 4 + k) * SB_N + v_kb * 128 + vg * 16) = o;
            }
          }
        }
      }
      fence_async_shared();
      mbar_arrive(&v_full[x]);
      load_v();
    }
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---- the rows of q: 8 rows x 4 pieces of 8 channels at a time
    const int quad = warp & 3, half = warp >> 2, c = lane & 3;
    float* rc = reinterpret_cast<float*>(smem + L::ROW);
#pragma unroll 1
    for (int r0 = warp * 16; r0 < warp * 16 + 16; r0 += 8) {
      const int row = r0 + (lane & 7), rr = tile * kTcRows + row;
      const int tok = (int)((uint32_t)rr / (uint32_t)a.r), hq = kvh * a.r + rr - tok * a.r;
      const float* qr = a.q + ((s.row0 + tok) * a.h + hq) * D + (lane >> 3) * 8;
      float y[NC][8], amax = 0.f, sum[NG];
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        float4 v0 = make_float4(0.f, 0.f, 0.f, 0.f), v1 = v0;
        if (row < rows) {
          v0 = *reinterpret_cast<const float4*>(qr + 32 * k);
          v1 = *reinterpret_cast<const float4*>(qr + 32 * k + 4);
        }
        y[k][0] = v0.x; y[k][1] = v0.y; y[k][2] = v0.z; y[k][3] = v0.w;
        y[k][4] = v1.x; y[k][5] = v1.y; y[k][6] = v1.z; y[k][7] = v1.w;
      }
#pragma unroll
      for (int n = 0; n < NG; ++n) sum[n] = 0.f;
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[k][i] *= a.scale2;
          amax = fmaxf(amax, fabsf(y[k][i]));
          sum[k * 32 / G] += y[k][i];
        }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 8));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 16));
      const int e = max(20, min(240, exp_field(amax)));
      const float up = pow2_field(268 - e);     // the largest magnitude in [2^14, 2^15)
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 8);
        sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 16);
        if (lane < 8) rc[(1 + n) * 128 + row] = sum[n] * up;
      }
      if (lane < 8) rc[row] = pow2_field(e - 14);
      uint8_t* qd = smem + L::Q + (row >> 3) * SB_D + (lane >> 3) * 128 + (lane & 7) * 16;
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        float h[8], l[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[k][i] *= up;
          h[i] = __half2float(__float2half_rn(y[k][i]));
          l[i] = y[k][i] - h[i];
        }
        *reinterpret_cast<uint4*>(qd + k * 512) =
            make_uint4(pack_h2(h[0], h[4]), pack_h2(h[2], h[6]), pack_h2(h[1], h[5]), pack_h2(h[3], h[7]));
        *reinterpret_cast<uint4*>(qd + kTcRows * D * 2 + k * 512) =
            make_uint4(pack_h2(l[0], l[4]), pack_h2(l[2], l[6]), pack_h2(l[1], l[5]), pack_h2(l[3], l[7]));
      }
    }
    fence_async_shared();
    mbar_arrive(q_full);
    named_barrier(2, 256 + 96);
    // all rows see the tiles up to here, and no block of theirs is missing
    const int all_there = s_missing ? INT32_MIN : all_see;
    // This lane: rows row0 and row0 + 8, of every 8 columns the pair 2 c, 2 c + 1.
    constexpr int NP = N / 8, OP = D / 8;
    const int row0 = quad * 32 + half * 16 + (lane >> 2);
    const uint32_t my_at = tmem + ((uint32_t)quad << 21) + ((uint32_t)half << 20);
    f2 qs[NG][2], rf[2], l2[2], mins[NG][2], o[OP][2];
    float m[2], corr[2] = {1.f, 1.f}, fac[NG] = {};
    int limit[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = row0 + 8 * i;
      rf[i] = pk(rc[row], rc[row]);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        qs[n][i] = pk(rc[(1 + n) * 128 + row], rc[(1 + n) * 128 + row]);
        mins[n][i] = 0;
      }
      l2[i] = 0;
      m[i] = -INFINITY;
      const int tok = (int)((uint32_t)(tile * kTcRows + row) / (uint32_t)a.r);
      limit[i] = row < rows ? max(0, min(s.len, s.len - s.n + tok + 1)) : 0;
    }
#pragma unroll
    for (int j = 0; j < OP; ++j) o[j][0] = o[j][1] = 0;
    bool ok = true;                             // after an expired wait the rounds go on without waits
    // the sums of values of tile t, added to what was there before
    auto flush = [&](int t) {
      const int x = t & 1;
      ok = __all_sync(0xffffffffu, ok && wait(&o_full[x], (uint32_t)(t >> 1) & 1u));
      if (!ok) return;
      tc_fence_after();
      if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f))
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f2 c2 = pk(corr[i], corr[i]);
#pragma unroll
          for (int j = 0; j < OP; ++j) o[j][i] = mul2(o[j][i], c2);
        }
      float acc[NS][32];
#pragma unroll
      for (int k = 0; k < NS; ++k) tmem_ld_frag(my_at + 256 + x * D + 64 * k, acc[k]);
      tmem_wait_ld();
#pragma unroll
      for (int k = 0; k < NS; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float f1 = fac[(64 * k + 8 * j) / G];
          const f2 f = pk(f1, f1);
          o[8 * k + j][0] = fma2(pk(acc[k][4 * j], acc[k][4 * j + 1]), f, o[8 * k + j][0]);
          o[8 * k + j][1] = fma2(pk(acc[k][4 * j + 2], acc[k][4 * j + 3]), f, o[8 * k + j][1]);
        }
      tc_fence_before();
    };
    constexpr int CH = N < 64 ? N : 64, CP = CH / 8;  // columns, pairs of a lane, of a TMEM access
    for (int t = 0; t < nt; ++t) {
      const int b2 = t & 1, slot = t % kPrmSlots, base = (t_first + t) * N + 2 * c;
      const float4* prm = reinterpret_cast<const float4*>(smem + L::PRM) + slot * 128 + c;
      ok = ok && wait(&prm_full[slot], (uint32_t)(t / kPrmSlots) & 1u) && wait(&s_full[b2], (uint32_t)(t >> 1) & 1u);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      const uint32_t s_at = my_at + b2 * 128;
      // x of 2 rows x NP pairs of tokens
      f2 x[NP][2];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float sc[N / CH][CP * 4];
#pragma unroll
        for (int k = 0; k < N / CH; ++k) tmem_ld_frag(s_at + n * N + k * CH, sc[k]);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < N / CH; ++k)
#pragma unroll
          for (int j = 0; j < CP; ++j) {
            const float4 p = prm[n * (N / 2) + 4 * (k * CP + j)];
            const f2 ks = pk(p.x, p.y), km = pk(p.z, p.w);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              f2& v = x[k * CP + j][i];
              const f2 b = n ? fma2(qs[n][i], km, v) : mul2(qs[n][i], km);
              v = fma2(pk(sc[k][4 * j + 2 * i], sc[k][4 * j + 2 * i + 1]), ks, b);
            }
          }
      }
      // what a row does not see, and what is not there
      const bool cut = (t_first + t + 1) * N > all_there;
      if (cut) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < NP; ++j)
            x[j][i] = pk(base + 8 * j < limit[i] ? lo_of(x[j][i]) : -INFINITY,
                         base + 8 * j + 1 < limit[i] ? hi_of(x[j][i]) : -INFINITY);
        // (the weights of these need nothing more: scale and minimum are 0)
        if (__builtin_expect(all_there == INT32_MIN, 0)) {
#pragma unroll
          for (int j = 0; j < NP; ++j)
            if (__float_as_uint(prm[4 * j].x) == 0x80000000u) x[j][0] = x[j][1] = pk(-INFINITY, -INFINITY);
        }
      }
      float keep[2];
      f2 ref2[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NP; ++j) top = fmaxf(top, fmaxf(lo_of(x[j][i]), hi_of(x[j][i])));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m_new = fmaxf(m[i], top * lo_of(rf[i]));
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        keep[i] = ex2(m[i] - ref);              // 0 while nothing was seen
        m[i] = m_new;
        ref2[i] = pk(-ref, -ref);
        const f2 k2 = pk(keep[i], keep[i]);
        l2[i] = mul2(l2[i], k2);
#pragma unroll
        for (int n = 0; n < NG; ++n) mins[n][i] = mul2(mins[n][i], k2);
      }
      // probabilities
      f2 more[2] = {0, 0};                      // a second chain of additions
#pragma unroll
      for (int j = 0; j < NP; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f2& v = x[j][i];
          v = fma2(v, rf[i], ref2[i]);
          v = pk(ex2(lo_of(v)), ex2(hi_of(v)));
          if (j & 1)
            more[i] = add2(more[i], v);
          else
            l2[i] = add2(l2[i], v);
        }
      l2[0] = add2(l2[0], more[0]);
      l2[1] = add2(l2[1], more[1]);
      // w in two terms over the scores, and the minima's sums
      auto weights = [&](auto part_seen) {
        constexpr bool kCut = decltype(part_seen)::value;
        const f2 minus = pk(-1.f, -1.f);
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int k = 0; k < N / CH; ++k) {
            uint32_t w[CP * 4];
#pragma unroll
            for (int jj = 0; jj < CP; ++jj) {
              const int j = k * CP + jj;
              const float4 p = prm[64 + n * (N / 2) + 4 * j];
              const f2 vs = pk(p.x, p.y), vm = pk(p.z, p.w);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                f2 w2 = mul2(x[j][i], vs);
                if (kCut) {                     // 0 times a NaN that this row does not see is 0
                  const bool in0 = base + 8 * j < limit[i], in1 = base + 8 * j + 1 < limit[i];
                  const f2 u = mul2(x[j][i], vm);
                  mins[n][i] = add2(mins[n][i], pk(in0 ? lo_of(u) : 0.f, in1 ? hi_of(u) : 0.f));
                  w2 = pk(in0 ? lo_of(w2) : 0.f, in1 ? hi_of(w2) : 0.f);
                } else {
                  mins[n][i] = fma2(x[j][i], vm, mins[n][i]);
                }
                // the high term is w cut to 11 bits (exact in fp16), the low one the rest
                const f2 high = w2 & 0xFFFFE000FFFFE000ull, rest = fma2(high, minus, w2);
                // 16 tokens: two groups of 4 columns of high terms, two of low ones
                uint32_t* d = &w[(jj >> 1) * 8 + (jj & 1) * 2 + i];
                d[0] = pack_h2(lo_of(high), hi_of(high));
                d[4] = pack_h2(lo_of(rest), hi_of(rest));
              }
            }
            tmem_st_frag(s_at + n * N + k * CH, w);
          }
      };
      if (cut)
        weights(std::true_type());
      else
        weights(std::false_type());
      float fac_new[NG];
#pragma unroll
      for (int n = 0; n < NG; ++n) fac_new[n] = reinterpret_cast<const float*>(smem + L::F)[slot * 4 + n];
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[b2]);
      if (t > 0) flush(t - 1);
      corr[0] = keep[0];
      corr[1] = keep[1];
#pragma unroll
      for (int n = 0; n < NG; ++n) fac[n] = fac_new[n];
    }
    if (nt > 0) flush(nt - 1);
    // ---- sums over the quad's lanes, and out
    const bool whole = splits == 1;
    float* part = reinterpret_cast<float*>(parts + (size_t)max(over, 0) * tc_part_floats(D) * 4);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = row0 + 8 * i;
      float l = lo_of(l2[i]) + hi_of(l2[i]), mn[NG];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        mn[n] = lo_of(mins[n][i]) + hi_of(mins[n][i]);
        mn[n] += __shfl_xor_sync(0xffffffffu, mn[n], 1);
        mn[n] += __shfl_xor_sync(0xffffffffu, mn[n], 2);
      }
      if (row < rows) {
        const int rr = tile * kTcRows + row;
        const int tok = (int)((uint32_t)rr / (uint32_t)a.r), hq = kvh * a.r + rr - tok * a.r;
        float* dst = (whole ? a.out + ((s.row0 + tok) * a.h + hq) * D : part + row * D) + 8 * c;
        const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int j = 0; j < OP; j += 4) {       // 4 nibbles x 2 lanes' g: 8 channels in a row
          float v[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[k] = (lo_of(o[j + k][i]) + mn[8 * j / G]) * inv;
            v[4 + k] = (hi_of(o[j + k][i]) + mn[8 * j / G]) * inv;
          }
          reinterpret_cast<float4*>(dst + 8 * j)[0] = make_float4(v[0], v[1], v[2], v[3]);
          reinterpret_cast<float4*>(dst + 8 * j)[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
        if (!whole && c == 0) {
          part[kTcRows * D + row] = m[i];
          part[kTcRows * (D + 1) + row] = l;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, kTmemCols);
}

template <int D, int NG>
int run(const Args& a, unsigned char* ws, cudaStream_t st) {
  using L = TcLayout<D, NG>;
  // a last wave of items or parts, whatever number of items it turns out to be
  const int64_t ctas = (tc_items(a) / a.sms + 1) * a.sms;
  NIMF_TRY(allow_smem((const void*)tc_kernel<D, NG>, L::SIZE));
  return launch(tc_kernel<D, NG>, dim3((unsigned)ctas), kTcThreads, L::SIZE, st, 1, a, ws);
}

}  // namespace

bool tc_serves(int d) { return d <= 128; }
size_t tc_ws_bytes(int d) { return ctx()->num_sms * tc_part_floats(d) * 4; }
int64_t tc_items(const Args& a) {
  const int64_t rows = a.rows * a.r;
  return (rows / kTcRows + std::min<int64_t>(a.n_seqs, rows / (a.big + 1))) * a.hkv;
}

int run_tc(const Args& a, int d, int ng, unsigned char* ws, cudaStream_t st) {
  switch (d * 16 + ng) {
    case 64 * 16 + 1: return run<64, 1>(a, ws, st);
    case 64 * 16 + 2: return run<64, 2>(a, ws, st);
    case 128 * 16 + 1: return run<128, 1>(a, ws, st);
    case 128 * 16 + 2: return run<128, 2>(a, ws, st);
    default: return run<128, 4>(a, ws, st);
  }
}

}  // namespace kv4
}  // namespace nimf
