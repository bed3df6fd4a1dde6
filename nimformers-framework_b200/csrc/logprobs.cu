// logprobs.cu -- log-probabilities of given tokens, their ranks, the entropy
// of each row of logits and its most likely tokens.
//
// With m = max x and the sums over all other entries
//   s = sum e^(x - m),  z = sum (x - m) e^(x - m):
//   log p(i) = (x_i - m) - log1p(s),   H = log1p(s) - z / (1 + s).
// The largest entry's own 1 stays out of s, so a row that is all but certain
// keeps the small probabilities that make up its entropy.
//
// The logits are read once: a cluster of CTAs holds one row in shared memory
// (bulk copies), and the passes over it (maxima, sums, candidates) stay there.
// The n-th largest of the threads' maxima is a lower bound of the row's n-th
// largest entry that few other entries reach, so the alternatives are chosen
// among little more than n candidates.
#include <cfloat>

#include "kv4.cuh"

namespace nimf {
namespace {

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kLpChunks = 4;      // bulk copies (and barriers) per slice
constexpr int kLpMaxTop = 32;
constexpr int kLpCand = 1024;     // candidates kept before the slow path
constexpr int kLpMaxCluster = 8;

struct LpPart {
  float m, s, z;                  // of one CTA's slice; s without the slice's maximum
  int nan, above;                 // a NaN in the slice; entries above the given logit
};

struct LpArgs {
  const float* x;
  const int32_t* ids;
  float* logprob;
  float* entropy;
  int32_t* rank;
  int32_t* top_ids;
  float* top_lp;
  int* err;
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

__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(const LpArgs a) {
  extern __shared__ __align__(128) float buf[];
  __shared__ uint64_t bar[kLpChunks];
  __shared__ float s_f[kLpWarps * 3];
  __shared__ int s_i[kLpWarps];
  __shared__ float s_sort[kLpWarps][32];
  __shared__ float c_v[kLpCand];
  __shared__ int c_i[kLpCand];
  __shared__ int c_n;
  __shared__ LpPart part[kLpMaxCluster];           // in the first CTA
  __shared__ float list_v[kLpMaxCluster * kLpMaxTop];
  __shared__ int list_i[kLpMaxCluster * kLpMaxTop];
  __shared__ float t_v[kLpMaxTop];                 // this CTA's alternatives
  __shared__ int t_i[kLpMaxTop];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned rank = kv4::cluster_rank(), ctas = kv4::cluster_size();
  const int64_t row = blockIdx.x / ctas;
  const int64_t lo = (int64_t)rank * a.slice;
  const int cnt = (int)max((int64_t)0, min((int64_t)a.slice, a.vocab - lo));
  griddep_launch_dependents();
  if (ctas > 1) kv4::cluster_arrive();             // met below, before remote stores
  if (tid == 0) {
    for (int i = 0; i < kLpChunks; ++i) mbar_init(&bar[i], 1);
    mbar_fence_init();
    c_n = 0;
  }
  __syncthreads();
  griddep_wait();

  // ---- the slice into shared memory, entry i at buf[pad + i]; the aligned
  // middle in bulk copies, the ends with plain loads, -inf around them
  const float* x = a.x + row * a.vocab + lo;
  const int pad = (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
  const int nf = (pad + cnt + 3) >> 2;             // float4s that hold entries
  const int mid0 = pad ? 1 : 0, mid1 = (pad + cnt) >> 2;   // whole ones
  const int per = ((nf + kLpChunks - 1) / kLpChunks + kLpThreads - 1) / kLpThreads * kLpThreads;
  if (tid == 0) {
    for (int i = 0; i < kLpChunks; ++i) {
      const int f0 = max(mid0, i * per), f1 = min(mid1, (i + 1) * per);
      const uint32_t bytes = f1 > f0 ? (uint32_t)(f1 - f0) * 16u : 0u;
      mbar_arrive_expect_tx(&bar[i], bytes);
      if (bytes) bulk_g2s(buf + 4 * f0, x + (4 * f0 - pad), bytes, &bar[i]);
    }
  }
  if (tid < 8) {
    // the first float4 if it is not whole, and the last one
    const int f = tid < 4 ? 0 : mid1;
    const bool mine = tid < 4 ? (mid0 == 1 || mid1 == 0) && nf > 0 : mid1 > 0 && mid1 < nf;
    if (mine) {
      const int i = 4 * f + (tid & 3) - pad;
      buf[4 * f + (tid & 3)] = i >= 0 && i < cnt ? x[i] : -INFINITY;
    }
  }
  const int64_t id = a.ids ? (int64_t)a.ids[row] : -1;
  const bool id_ok = id >= 0 && id < a.vocab;
  const float given = id_ok ? a.x[row * a.vocab + id] : INFINITY;
  __syncthreads();

  // ---- maxima, and the entries above the given one
  const float4* b4 = reinterpret_cast<const float4*>(buf);
  float tm = -INFINITY;
  int above = 0;
  bool ok = true;
  for (int i = 0; i < kLpChunks; ++i) {
    ok = ok && mbar_wait_t<0>(&bar[i], 0);
    const int f1 = min(nf, (i + 1) * per);
    for (int f = i * per + tid; f < f1; f += kLpThreads) {
      const float4 v = b4[f];
      tm = fmaxf(fmaxf(tm, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
      above += (v.x > given) + (v.y > given) + (v.z > given) + (v.w > given);
    }
  }
  if (!ok && a.err) atomicExch(a.err, 6);
  float m = tm;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    above += __shfl_xor_sync(0xffffffffu, above, o);
  }
  if (lane == 0) {
    s_f[warp] = m;
    s_i[warp] = above;
  }
  __syncthreads();
  m = s_f[0];
  above = s_i[0];
  for (int i = 1; i < kLpWarps; ++i) {
    m = fmaxf(m, s_f[i]);
    above += s_i[i];
  }
  __syncthreads();

  // ---- sums; only a thread that holds the maximum has to look for it
  float s = 0.f, z = 0.f;
  int at_max = 0, nan = 0;
  if (m == -INFINITY) {
    for (int f = tid; f < nf; f += kLpThreads) {
      const float4 v = b4[f];
      nan |= v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w;
    }
  } else if (tm == m) {
    for (int f = tid; f < nf; f += kLpThreads) {
      const float4 v = b4[f];
      const float e4[4] = {v.x, v.y, v.z, v.w};
      for (int e = 0; e < 4; ++e) {
        if (e4[e] == m) {
          ++at_max;
          if (m == INFINITY) s = __int_as_float(0x7fffffff);
        } else {
          float t = e4[e] - m;
          const float w = exp_term(t);
          s += w;
          z = fmaf(t, w, z);
        }
      }
    }
  } else {
    float s1 = 0.f, z1 = 0.f;
    for (int f = tid; f < nf; f += kLpThreads) {
      const float4 v = b4[f];
      float t0 = v.x - m, t1 = v.y - m, t2 = v.z - m, t3 = v.w - m;
      const float w0 = exp_term(t0), w1 = exp_term(t1), w2 = exp_term(t2), w3 = exp_term(t3);
      s += w0 + w1;
      s1 += w2 + w3;
      z = fmaf(t0, w0, fmaf(t1, w1, z));
      z1 = fmaf(t2, w2, fmaf(t3, w3, z1));
    }
    s += s1;
    z += z1;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    z += __shfl_xor_sync(0xffffffffu, z, o);
    nan |= __shfl_xor_sync(0xffffffffu, nan, o);
  }
  // every entry equal to the maximum counts 1, but for the first one
  const unsigned holders = __ballot_sync(0xffffffffu, at_max > 0);
  const bool first_holder = holders && lane == __ffs(holders) - 1;
  if (lane == 0) s_i[warp] = holders != 0;
  __syncthreads();
  bool earlier = false;
  for (int i = 0; i < warp; ++i) earlier |= s_i[i] != 0;
  s += (float)(at_max - (first_holder && !earlier ? 1 : 0));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) {
    s_f[warp] = s;
    s_f[kLpWarps + warp] = z;
    s_f[2 * kLpWarps + warp] = nan ? 1.f : 0.f;
  }
  __syncthreads();
  LpPart mine = {m, 0.f, 0.f, 0, above};
  for (int i = 0; i < kLpWarps; ++i) {
    mine.s += s_f[i];
    mine.z += s_f[kLpWarps + i];
    mine.nan |= s_f[2 * kLpWarps + i] != 0.f;
  }

  // ---- the slice's alternatives
  const int top = a.top;
  if (top > 0) {
    // the top-th largest of the threads' maxima
    float v = warp_sort(tm);
    for (int half = kLpWarps / 2; half > 0; half >>= 1) {
      if (warp >= half && warp < 2 * half) s_sort[warp][lane] = v;
      __syncthreads();
      if (warp < half) v = warp_merge(v, s_sort[warp + half][31 - lane]);
    }
    if (warp == 0) s_sort[0][lane] = v;
    __syncthreads();
    const float bound = s_sort[0][top - 1];
    if (tm >= bound && tm > -INFINITY)
      for (int f = tid; f < nf; f += kLpThreads) {
        const float4 v4 = b4[f];
        const float e4[4] = {v4.x, v4.y, v4.z, v4.w};
        for (int e = 0; e < 4; ++e)
          if (e4[e] >= bound && e4[e] > -INFINITY) {
            const int k = atomicAdd(&c_n, 1);
            if (k < kLpCand) {
              c_v[k] = e4[e];
              c_i[k] = 4 * f + e - pad;
            }
          }
      }
    __syncthreads();
    int n = c_n;
    const int want = min(top, cnt);
    if (n <= kLpCand) {
      for (int i = tid; i < n; i += kLpThreads) {
        const float w = c_v[i];
        const int wi = c_i[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += before(c_v[j], c_i[j], w, wi);
        if (r < want) {
          t_v[r] = w;
          t_i[r] = wi;
        }
      }
      // fewer entries above -inf than asked for: the first of the others
      if (n < want && warp == 0) {
        for (int i0 = 0; n < want && i0 < cnt; i0 += 32) {
          const int i = i0 + lane;
          const bool rest = i < cnt && !(buf[pad + i] > -INFINITY);
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
          const float4 v4 = b4[f];
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
      const uint32_t w[5] = {__float_as_uint(mine.m), __float_as_uint(mine.s), __float_as_uint(mine.z),
                             (uint32_t)mine.nan, (uint32_t)mine.above};
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
    // sums over the slices, in their order
    float M = -INFINITY;
    int who = -1;
    for (unsigned i = 0; i < ctas; ++i) {
      if (part[i].m > M) {
        M = part[i].m;
        who = (int)i;
      }
    }
    LpPart all = {M, 0.f, 0.f, 0, 0};
    for (unsigned i = 0; i < ctas; ++i) {
      all.nan |= part[i].nan;
      all.above += part[i].above;
      if (part[i].m == -INFINITY) continue;
      float d = part[i].m - M;
      const float d0 = d, f = (int)i == who ? 1.f : exp_term(d);
      const float tot = 1.f + part[i].s;
      all.s += (int)i == who ? part[i].s : f * tot;
      all.z += (int)i == who ? part[i].z : f * fmaf(max_nan(d0, -128.f), tot, part[i].z);
    }
    mine = all;
    const int n = (int)ctas * top;
    for (int i = tid; i < n; i += kLpThreads) {
      const float w = list_v[i];
      const int wi = list_i[i];
      if (wi == INT32_MAX) continue;
      int r = 0;
      for (int j = 0; j < n; ++j) r += before(list_v[j], list_i[j], w, wi);
      if (r < top) {
        t_v[r] = w;
        t_i[r] = wi;
      }
    }
    __syncthreads();
  }

  const float nanf_ = __int_as_float(0x7fffffff);
  const bool empty = mine.m == -INFINITY;          // nothing is possible
  const float log_s = log1pf(mine.s);
  auto lp = [&](float w) -> float {
    if (mine.nan) return nanf_;
    return empty ? -INFINITY : (w - mine.m) - log_s;
  };
  if (tid < top) {
    a.top_ids[row * top + tid] = t_i[tid];
    a.top_lp[row * top + tid] = lp(t_v[tid]);
  }
  if (tid == 0) {
    if (a.logprob) a.logprob[row] = id_ok ? lp(given) : mine.nan || mine.s != mine.s ? nanf_ : -INFINITY;
    if (a.entropy) a.entropy[row] = mine.nan ? nanf_ : empty ? 0.f : log_s - mine.z / (1.f + mine.s);
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
  // As many CTAs a row as bring its slice to 16,384 entries (three CTAs to an
  // SM then), more where few rows would leave SMs without work.
  unsigned ctas = 1;
  while (ctas < (unsigned)kLpMaxCluster &&
         ((vocab + ctas - 1) / ctas > 16384 ||
          (rows * ctas < ctx()->num_sms && vocab / ctas > 4 * kLpThreads)))
    ctas *= 2;
  LpArgs a = {};
  a.x = logits;
  a.ids = ids;
  a.logprob = logprob;
  a.entropy = entropy;
  a.rank = rank;
  a.top_ids = top_ids;
  a.top_lp = top_logprobs;
  a.err = ctx()->dev_err;
  a.vocab = vocab;
  a.slice = (int)(((vocab + ctas - 1) / ctas + 3) & ~(int64_t)3);
  a.top = (int)n_top;
  const size_t smem = (size_t)(a.slice + 8) * 4;
  NIMF_TRY(kv4::allow_smem((const void*)logprobs_kernel, 160 * 1024));
  return kv4::launch(logprobs_kernel, dim3((unsigned)(rows * ctas)), kLpThreads, smem, st, ctas, a);
}
