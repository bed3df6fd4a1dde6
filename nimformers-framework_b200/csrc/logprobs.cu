// logprobs.cu -- log-probabilities of given tokens, their ranks, the entropy
// of each row of logits and its most likely tokens.
//
// With m = max x and the sums over all other entries
//   s = sum e^(x - m),  z = sum (x - m) e^(x - m):
//   log p(i) = (x_i - m) - log1p(s),   H = log1p(s) - z / (1 + s).
// The largest entry's own 1 stays out of s, so a row that is all but certain
// keeps the small probabilities that make up its entropy.
//
// The logits are read once from HBM: a thread streams its share with a running
// maximum and sums (four float4 loads ahead of their use), a CTA takes a row, a
// cluster of CTAs shares one where rows are few or long.  The n-th largest of the
// threads' maxima is a lower bound of the row's n-th largest entry that few other
// entries reach, so the alternatives are chosen among little more than n
// candidates, for which the threads that reach the bound read their shares again
// (out of L2).  Bounded by HBM; a slice kept in shared memory instead cost 64 KB
// a CTA, loads and passes took turns, and 4,096 rows of 32,000 took 230 us; they
// take 92 us now (5.7 TB/s; 102 us with buffers of its own for every call), 64 rows
// of 128,001 with 20 alternatives 12.5 us, one row of 32,000 6.2 us, both of these
// latency (times of captured calls).
#include <cfloat>

#include "kv4.cuh"

namespace nimf {
namespace {

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kLpAhead = 4;       // float4s of a thread in flight
constexpr int kLpMaxTop = 32;
constexpr int kLpCand = 1024;     // candidates kept before the slow path
constexpr int kLpMaxCluster = 8;

// Entries seen, relative to a reference r >= all of them: top = e^(max - r), the
// sum s of all other terms and z of all (x - r) e^(x - r).  Whatever is added,
// the smaller of two tops joins s and the larger stays out of it, so at the end,
// where r is the maximum and top is 1, s holds exactly the other entries.  z is
// NaN once a NaN or +inf was seen.
struct LpPart {
  float r, top, s, z;
  int above;                      // entries above the given logit
};

struct LpArgs {
  const float* x;
  const int32_t* ids;
  float* logprob;
  float* entropy;
  int32_t* rank;
  int32_t* top_ids;
  float* top_lp;
  int64_t vocab;
  int slice, top;
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// e^t for t <= 0 (t = NaN gives NaN); t below -128 gives 0, so that t e^t is 0
// for t = -inf too.
__device__ __forceinline__ float exp_term(float& t) {
  t = max_nan(t, -128.f);
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t * 1.44269504f));
  return e;
}

// Moves the reference up to r (r = -inf: nothing seen, all sums are 0).
__device__ __forceinline__ void lp_raise(LpPart& a, float r) {
  if (r == a.r) return;
  if (a.r > -INFINITY) {
    float d = a.r - r;
    const float f = exp_term(d);
    a.z = f * fmaf(d, a.s + a.top, a.z);
    a.s *= f;
    a.top *= f;
  }
  a.r = r;
}
__device__ __forceinline__ void lp_add(LpPart& a, float top, float s, float z) {
  a.s += s + fminf(a.top, top);
  a.top = fmaxf(a.top, top);
  a.z += z;
}

// The parts of disjoint sets, in their order.
__device__ __forceinline__ LpPart lp_join(const LpPart* p, int n) {
  float r = p[0].r;
  for (int i = 1; i < n; ++i) r = fmaxf(r, p[i].r);
  LpPart all = p[0];
  lp_raise(all, r);
  for (int i = 1; i < n; ++i) {
    LpPart b = p[i];
    lp_raise(b, r);
    lp_add(all, b.top, b.s, b.z);
    all.above += b.above;
  }
  return all;
}

// Falling order over the warp's lanes of one float each.
__device__ __forceinline__ float warp_sort(float v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const float u = __shfl_xor_sync(0xffffffffu, v, j);
      const bool keep_max = ((lane & j) == 0) == ((lane & k) == 0);
      v = keep_max ? fmaxf(v, u) : fminf(v, u);
    }
  return v;
}
// The 32 largest of two falling lists of 32, falling.
__device__ __forceinline__ float warp_merge(float v, float other_reversed) {
  const int lane = threadIdx.x & 31;
  v = fmaxf(v, other_reversed);
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, j);
    v = (lane & j) == 0 ? fmaxf(v, u) : fminf(v, u);
  }
  return v;
}

__device__ __forceinline__ uint32_t remote_smem(const void* p, unsigned cta) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(cta));
  return r;
}
__device__ __forceinline__ void st_remote(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Whether (v, i) comes before (w, j) among the alternatives.
__device__ __forceinline__ bool before(float v, int i, float w, int j) {
  return v > w || (v == w && i < j);
}

// A slice of a row as float4s: entry i is element i + pad of them.
struct LpSlice {
  const float* x;                 // 16-byte aligned: pad entries before the slice
  int pad, cnt, nf;
  __device__ __forceinline__ float4 load_whole(int f) const {
    float4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "l"(x + 4 * (int64_t)f));
    return v;
  }
  __device__ __forceinline__ float4 load(int f) const {
    const int i = 4 * f - pad;
    if (i >= 0 && i + 4 <= cnt) return load_whole(f);
    float4 v;                     // an end of the slice, or nothing
    const float* p = x + 4 * (int64_t)f;
    v.x = i >= 0 && i < cnt ? p[0] : -INFINITY;
    v.y = i + 1 >= 0 && i + 1 < cnt ? p[1] : -INFINITY;
    v.z = i + 2 >= 0 && i + 2 < cnt ? p[2] : -INFINITY;
    v.w = i + 3 >= 0 && i + 3 < cnt ? p[3] : -INFINITY;
    return v;
  }
};

// How many of n entries (rounded up to four; what is there counts) come before (w, wi).
__device__ __forceinline__ int rank_of(const float* v, const int* i, int n, float w, int wi) {
  int r = 0;
#pragma unroll 4
  for (int j = 0; j < n; j += 4) {
    const float4 a = *reinterpret_cast<const float4*>(v + j);
    const int4 b = *reinterpret_cast<const int4*>(i + j);
    r += before(a.x, b.x, w, wi) + before(a.y, b.y, w, wi) + before(a.z, b.z, w, wi) + before(a.w, b.w, w, wi);
  }
  return r;
}

// PER_SM CTAs fit an SM.  Two, with all the registers that they want, where all of
// the grid runs at once (64 rows of 128,001 in clusters of 4: 12.5 us, 15.3 with
// three, 17.4 with four; 200 rows of 32,000: 9.6, with four 15.9); four where rows
// queue (4,096 rows of 32,000: 92 us, 102 with three, 98 with five, which spill).
template <int PER_SM>
__global__ void __launch_bounds__(kLpThreads, PER_SM) logprobs_kernel(const LpArgs a) {
  __shared__ LpPart s_part[kLpWarps];
  __shared__ float s_f[kLpWarps];
  __shared__ int s_i[kLpWarps];
  __shared__ float s_sort[kLpWarps][32];
  __shared__ __align__(16) float c_v[kLpCand];
  __shared__ __align__(16) int c_i[kLpCand];
  __shared__ int c_n, s_n;
  __shared__ int s_who[kLpThreads];                // threads whose share holds candidates
  __shared__ LpPart part[kLpMaxCluster];           // in the first CTA
  __shared__ __align__(16) float list_v[kLpMaxCluster * kLpMaxTop];
  __shared__ __align__(16) int list_i[kLpMaxCluster * kLpMaxTop];
  __shared__ float t_v[kLpMaxTop];                 // this CTA's alternatives
  __shared__ int t_i[kLpMaxTop];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned rank = kv4::cluster_rank(), ctas = kv4::cluster_size();
  const int64_t row = blockIdx.x / ctas;
  const int64_t lo = (int64_t)rank * a.slice;
  LpSlice sl;
  sl.cnt = (int)max((int64_t)0, min((int64_t)a.slice, a.vocab - lo));
  griddep_launch_dependents();
  if (ctas > 1) kv4::cluster_arrive();             // met below, before remote stores
  if (tid == 0) c_n = s_n = 0;
  griddep_wait();
  const float* x = a.x + row * a.vocab + lo;
  sl.pad = (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
  sl.x = x - sl.pad;
  sl.nf = (sl.pad + sl.cnt + 3) >> 2;
  const int cnt = sl.cnt, pad = sl.pad, nf = sl.nf;
  const int64_t id = a.ids ? (int64_t)a.ids[row] : -1;
  const bool id_ok = id >= 0 && id < a.vocab;
  const float given = id_ok ? a.x[row * a.vocab + id] : INFINITY;

  // ---- one pass: maximum, sums, entries above the given one
  LpPart me = {-INFINITY, 0.f, 0.f, 0.f, 0};
  float tm = -INFINITY;                            // this thread's largest entry
  {
    constexpr int kRound = kLpAhead * kLpThreads;  // float4s of a round of the CTA
    const int whole = (pad + cnt) >> 2;            // those before are full, but for the first
    auto fetch = [&](int f0, float4 (&v)[kLpAhead]) {
      if (f0 + kRound <= whole && (f0 > 0 || pad == 0)) {
#pragma unroll
        for (int k = 0; k < kLpAhead; ++k) v[k] = sl.load_whole(f0 + tid + k * kLpThreads);
      } else {
#pragma unroll
        for (int k = 0; k < kLpAhead; ++k) v[k] = sl.load(f0 + tid + k * kLpThreads);
      }
    };
    auto take = [&](const float4 (&v)[kLpAhead]) {
      float e[4 * kLpAhead];
#pragma unroll
      for (int k = 0; k < kLpAhead; ++k) {
        e[4 * k] = v[k].x;
        e[4 * k + 1] = v[k].y;
        e[4 * k + 2] = v[k].z;
        e[4 * k + 3] = v[k].w;
      }
      float most = e[0];
#pragma unroll
      for (int k = 0; k < 4 * kLpAhead; ++k) {
        most = fmaxf(most, e[k]);                  // a NaN has no say
        me.above += e[k] > given;
      }
      tm = fmaxf(tm, most);
      // one reference a warp: no lane leaves the common path
      float all;
      asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(all) : "f"(most));
      if (all > me.r) lp_raise(me, all);
      const float ref = me.r == -INFINITY ? 0.f : me.r;
      float s1 = 0.f, z1 = 0.f, top1 = 0.f;        // a second chain
#pragma unroll
      for (int k = 0; k < 4 * kLpAhead; ++k) {
        float t = e[k] - ref;
        const float w = exp_term(t);
        float& top = k & 1 ? top1 : me.top;
        (k & 1 ? s1 : me.s) += fminf(top, w);
        top = fmaxf(top, w);
        float& z = k & 1 ? z1 : me.z;
        z = fmaf(t, w, z);
      }
      lp_add(me, top1, s1, z1);
    };
    // two rounds' registers in turn
    float4 va[kLpAhead], vb[kLpAhead];
    fetch(0, va);
#pragma unroll 1
    for (int f0 = 0; f0 < nf; f0 += 2 * kRound) {
      if (f0 + kRound < nf) fetch(f0 + kRound, vb);
      take(va);
      if (f0 + kRound < nf) {
        if (f0 + 2 * kRound < nf) fetch(f0 + 2 * kRound, va);
        take(vb);
      }
    }
  }
  LpPart mine = me;                                // the lanes have one reference
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lp_add(mine, __shfl_xor_sync(0xffffffffu, mine.top, o), __shfl_xor_sync(0xffffffffu, mine.s, o),
           __shfl_xor_sync(0xffffffffu, mine.z, o));
    mine.above += __shfl_xor_sync(0xffffffffu, mine.above, o);
  }
  if (lane == 0) s_part[warp] = mine;
  __syncthreads();
  mine = lp_join(s_part, kLpWarps);

  // ---- the slice's alternatives
  const int top = a.top;
  if (top > 0) {
    // the top-th largest of the threads' maxima
    float bound;
    if (top == 1) {
      bound = mine.r;                              // the slice's maximum
    } else {
      float v = warp_sort(tm);
      for (int half = kLpWarps / 2; half > 0; half >>= 1) {
        if (warp >= half && warp < 2 * half) s_sort[warp][lane] = v;
        __syncthreads();
        if (warp < half) v = warp_merge(v, s_sort[warp + half][31 - lane]);
      }
      if (warp == 0) s_sort[0][lane] = v;
      __syncthreads();
      bound = s_sort[0][top - 1];
    }
    // the threads that reach it, and their shares again, a warp a share
    if (tm >= bound && tm > -INFINITY) s_who[atomicAdd(&s_n, 1)] = tid;
    __syncthreads();
    for (int k = warp; k < s_n; k += 4 * kLpWarps)
      for (int f0 = lane * kLpThreads; f0 - lane * kLpThreads < nf; f0 += 32 * kLpThreads) {
        float4 v[4];                               // of four shares
        int f[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f[q] = k + q * kLpWarps < s_n ? f0 + s_who[k + q * kLpWarps] : nf;
          v[q] = sl.load(f[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float e4[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e4[e] >= bound && e4[e] > -INFINITY) {
              const int at = atomicAdd(&c_n, 1);
              if (at < kLpCand) {
                c_v[at] = e4[e];
                c_i[at] = 4 * f[q] + e - pad;
              }
            }
        }
      }
    __syncthreads();
    if (tid < 4 && c_n + tid < kLpCand) {          // whole fours for the comparisons
      c_v[c_n + tid] = -INFINITY;
      c_i[c_n + tid] = INT32_MAX;
    }
    __syncthreads();
    int n = c_n;
    const int want = min(top, cnt);
    if (n <= kLpCand) {
      for (int i = tid; i < n; i += kLpThreads) {
        const float w = c_v[i];
        const int wi = c_i[i];
        const int r = rank_of(c_v, c_i, n, w, wi);
        if (r < want) {
          t_v[r] = w;
          t_i[r] = wi;
        }
      }
      // fewer entries above -inf than asked for: the first of the others
      if (n < want && warp == 0) {
        for (int i0 = 0; n < want && i0 < cnt; i0 += 32) {
          const int i = i0 + lane;
          const bool rest = i < cnt && !(x[i] > -INFINITY);
          const unsigned who = __ballot_sync(0xffffffffu, rest);
          const int r = n + __popc(who & ((1u << lane) - 1u));
          if (rest && r < want) {
            t_v[r] = -INFINITY;
            t_i[r] = i;
          }
          n += __popc(who);
        }
      }
    } else {
      // Many entries equal (or as good as sorted): one entry a round, the
      // first after the last one chosen.
      float pv = INFINITY;
      int pi = -1;
      for (int r = 0; r < want; ++r) {
        float bv = -INFINITY;
        int bi = INT32_MAX;
        for (int f = tid; f < nf; f += kLpThreads) {
          const float4 v4 = sl.load(f);
          const float e4[4] = {v4.x, v4.y, v4.z, v4.w};
          for (int e = 0; e < 4; ++e) {
            const int i = 4 * f + e - pad;
            if (i < 0 || i >= cnt) continue;
            const float w = e4[e] == e4[e] ? e4[e] : -INFINITY;
            if ((r == 0 || before(pv, pi, w, i)) && before(w, i, bv, bi)) {
              bv = w;
              bi = i;
            }
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const float u = __shfl_xor_sync(0xffffffffu, bv, o);
          const int ui = __shfl_xor_sync(0xffffffffu, bi, o);
          if (before(u, ui, bv, bi)) {
            bv = u;
            bi = ui;
          }
        }
        if (lane == 0) {
          s_f[warp] = bv;
          s_i[warp] = bi;
        }
        __syncthreads();
        pv = s_f[0];
        pi = s_i[0];
        for (int i = 1; i < kLpWarps; ++i)
          if (before(s_f[i], s_i[i], pv, pi)) {
            pv = s_f[i];
            pi = s_i[i];
          }
        if (tid == 0) {
          t_v[r] = pv;
          t_i[r] = pi;
        }
        __syncthreads();
      }
    }
    __syncthreads();
  }

  // ---- the slices of a row meet in the cluster's first CTA
  if (ctas > 1) {
    kv4::cluster_wait();
    if (tid < 5) {
      const uint32_t w[5] = {__float_as_uint(mine.r), __float_as_uint(mine.top), __float_as_uint(mine.s),
                             __float_as_uint(mine.z), (uint32_t)mine.above};
      st_remote(remote_smem(&part[rank], 0) + tid * 4, w[tid]);
    }
    if (tid < top) {
      const bool has = tid < cnt;
      st_remote(remote_smem(&list_v[rank * top + tid], 0), __float_as_uint(has ? t_v[tid] : -INFINITY));
      st_remote(remote_smem(&list_i[rank * top + tid], 0),
                (uint32_t)(has ? (int)lo + t_i[tid] : INT32_MAX));
    }
    kv4::cluster_arrive();
    kv4::cluster_wait();
    if (rank != 0) return;
    if (tid < 4 && (int)ctas * top + tid < kLpMaxCluster * kLpMaxTop) {
      list_v[ctas * top + tid] = -INFINITY;
      list_i[ctas * top + tid] = INT32_MAX;
    }
    __syncthreads();
    // sums over the slices, in their order
    mine = lp_join(part, (int)ctas);
    const int n = (int)ctas * top;
    for (int i = tid; i < n; i += kLpThreads) {
      const float w = list_v[i];
      const int wi = list_i[i];
      if (wi == INT32_MAX) continue;
      const int r = rank_of(list_v, list_i, n, w, wi);
      if (r < top) {
        t_v[r] = w;
        t_i[r] = wi;
      }
    }
    __syncthreads();
  }

  const float nanf_ = __int_as_float(0x7fffffff);
  const bool bad = mine.z != mine.z, empty = mine.r == -INFINITY;  // NaN or +inf; nothing is possible
  const float log_s = log1pf(mine.s);
  auto lp = [&](float w) -> float { return bad ? nanf_ : empty ? -INFINITY : (w - mine.r) - log_s; };
  if (tid < top) {
    a.top_ids[row * top + tid] = t_i[tid];
    a.top_lp[row * top + tid] = lp(t_v[tid]);
  }
  if (tid == 0) {
    if (a.logprob) a.logprob[row] = id_ok ? lp(given) : bad ? nanf_ : -INFINITY;
    if (a.entropy) a.entropy[row] = bad ? nanf_ : empty ? 0.f : log_s - mine.z / (1.f + mine.s);
    if (a.rank) a.rank[row] = id_ok ? mine.above + 1 : 0;
  }
}

}  // namespace
}  // namespace nimf

using namespace nimf;

extern "C" int nimf_logprobs_dev(const float* logits, int64_t rows, int64_t vocab,
                                 const int32_t* ids, int64_t n_top, float* logprob, float* entropy,
                                 int32_t* rank, int32_t* top_ids, float* top_logprobs,
                                 void* stream) {
  cudaStream_t st;
  const int64_t max_vocab = (int64_t)32 * 1024 * 8;
  if (rows < 0 || rows > INT32_MAX / kLpMaxCluster || vocab < 1 || vocab > max_vocab || n_top < 0 ||
      n_top > kLpMaxTop || n_top > vocab)
    return set_error(NIMF_ERR_SHAPE, "logprobs: rows %lld vocab %lld (1..%lld) n_top %lld (<= %d, <= vocab)",
                     (long long)rows, (long long)vocab, (long long)max_vocab, (long long)n_top, kLpMaxTop);
  if (rows == 0) return NIMF_OK;
  if (!logits || ((logprob || rank) && !ids) || (n_top > 0 && (!top_ids || !top_logprobs)))
    return set_error(NIMF_ERR_ARG, "logprobs: NULL buffer");
  NIMF_TRY(kv4::stream_of(stream, &st));
  // A CTA a row; several where the rows do not fill the SMs, up to two CTAs an SM,
  // as long as a thread keeps two float4s.
  unsigned ctas = 1;
  while (ctas < (unsigned)kLpMaxCluster && rows * ctas <= ctx()->num_sms && vocab / ctas > 4 * kLpThreads * kLpAhead)
    ctas *= 2;
  LpArgs a = {};
  a.x = logits;
  a.ids = ids;
  a.logprob = logprob;
  a.entropy = entropy;
  a.rank = rank;
  a.top_ids = top_ids;
  a.top_lp = top_logprobs;
  a.vocab = vocab;
  a.slice = (int)(((vocab + ctas - 1) / ctas + 3) & ~(int64_t)3);
  a.top = (int)n_top;
  return kv4::launch(rows * ctas <= 2 * ctx()->num_sms ? logprobs_kernel<2> : logprobs_kernel<4>, dim3((unsigned)(rows * ctas)), kLpThreads, 0, st, ctas, a);
}
