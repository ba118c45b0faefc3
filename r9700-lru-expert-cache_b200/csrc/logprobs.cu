// Log probabilities of given tokens from logits [M, V], with entropy, rank and top alternatives.
//
// One pass over a row. A thread walks 16-byte chunks of it (8 or 4 logits), keeping sums relative to a
// reference m that it takes from the first logits it sees and moves only when one exceeds it by 40:
//   S = sum 2^y,  W = sum 2^y y,  y = (x - m) log2 e,  and n = #{x > x_t};
// references differ between threads and meet at the end: moving a part to a larger M is S 2^t and
// (W + S t) 2^t, t = (m - M) log2 e. With M the maximum, ln S and W / S give everything but the order.
//
// The top alternatives cost the pass nothing but each thread's maximum and where it first was. The k-th
// largest of any k or more disjoint groups' maxima bounds the k-th largest logit from below, so only the
// few threads whose maximum reaches it can hold a top logit: their chunks are read again, and the handful
// of logits at or above the bound is ordered by counting. Order is (value descending, id ascending) as one
// 64-bit key, so nothing depends on timing.
//
// A row is shared by a cluster of 1 to 8 CTAs, so that few rows still occupy the SMs.
#include <algorithm>

#include "score.cuh"
#include "tcgen05.cuh"

namespace {

using namespace b200;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int MAX_TOP = 64;
constexpr int GROUPS = 64;                 // at least MAX_TOP disjoint groups of a CTA's threads
constexpr int CAND = 1024;                 // logits at or above the bound that are kept; more take the slow way
constexpr int INFLIGHT = 4;                // chunks a thread loads at a time
constexpr float HEADROOM = 40.f;           // e^40 times the vocabulary stays far below fp32's largest

template <typename T>
struct Chunk;                              // 16 bytes of logits

template <>
struct Chunk<float> {
  static constexpr int N = 4;
  static constexpr bool PACKED = false;
  __device__ static float value(const uint4& c, int i) {
    return __uint_as_float(i == 0 ? c.x : i == 1 ? c.y : i == 2 ? c.z : c.w);
  }
  __device__ static float top(const uint4& c) {
    return max_nan(max_nan(value(c, 0), value(c, 1)), max_nan(value(c, 2), value(c, 3)));
  }
  __device__ static float of(float v) { return v; }
};

__device__ __forceinline__ uint32_t word(const uint4& c, int i) { return i == 0 ? c.x : i == 1 ? c.y : i == 2 ? c.z : c.w; }

template <>
struct Chunk<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr bool PACKED = true;
  using Pair = __nv_bfloat162;
  __device__ static Pair pair(const uint4& c, int i) {
    const uint32_t w = word(c, i);
    return *reinterpret_cast<const Pair*>(&w);
  }
  __device__ static float value(const uint4& c, int i) {
    const uint32_t w = word(c, i >> 1);
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
  __device__ static float top(const uint4& c) {
    const Pair m = __hmax2_nan(__hmax2_nan(pair(c, 0), pair(c, 1)), __hmax2_nan(pair(c, 2), pair(c, 3)));
    return max_nan(__low2float(m), __high2float(m));
  }
  __device__ static float of(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static Pair both(float v) { return __float2bfloat162_rn(v); }
};

template <>
struct Chunk<__half> {
  static constexpr int N = 8;
  static constexpr bool PACKED = true;
  using Pair = __half2;
  __device__ static Pair pair(const uint4& c, int i) {
    const uint32_t w = word(c, i);
    return *reinterpret_cast<const Pair*>(&w);
  }
  __device__ static float value(const uint4& c, int i) {
    const Pair p = pair(c, i >> 1);
    return i & 1 ? __high2float(p) : __low2float(p);
  }
  __device__ static float top(const uint4& c) {
    const Pair m = __hmax2_nan(__hmax2_nan(pair(c, 0), pair(c, 1)), __hmax2_nan(pair(c, 2), pair(c, 3)));
    return max_nan(__low2float(m), __high2float(m));
  }
  __device__ static float of(__half v) { return __half2float(v); }
  __device__ static Pair both(float v) { return __float2half2_rn(v); }
};

// Order of (value, id) as one whole number: the larger value first, then the lower id. NaN above +inf, -0 equal
// to +0.
__device__ __forceinline__ unsigned long long order_key(float x, int id) {
  uint32_t u = __float_as_uint(x + 0.f);
  u = isnan(x) ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (uint32_t)~id;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// (a.x + b.x, a.y + b.y), (a.x b.x, a.y b.y) and a fused multiply-add, one packed instruction each.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
        "l"(*reinterpret_cast<unsigned long long*>(&c)));
  return *reinterpret_cast<float2*>(&r);
}

// What the CTAs of a row's cluster leave for its first one.
struct Part {
  float m, s, w;                           // natural maximum; S and W in units of log2 e
  int above, n_top;
  unsigned long long top[MAX_TOP];
};

struct Args {
  const void* logits;
  long long ld;
  int V;
  const long long* ids;
  int top_k;
  float* logprob;
  long long* rank;
  float* entropy;
  float* lse;
  long long* top_ids;
  float* top_lp;
};

template <typename T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_logprobs_kernel(Args p) {
  using C = Chunk<T>;
  constexpr int N = C::N, WARPS = THREADS / 32;
  __shared__ Part part;
  __shared__ float sh_m[WARPS], sh_s[WARPS], sh_w[WARPS];
  __shared__ int sh_n[WARPS];
  __shared__ unsigned long long keys[TOP ? THREADS : 1], group_key[TOP ? GROUPS : 1], cand[TOP ? CAND : 1];
  __shared__ int list[TOP ? THREADS : 1];
  __shared__ int n_list, n_cand;
  __shared__ unsigned long long bound_s;
  const int crank = (int)cluster_rank(), csize = (int)cluster_size();
  const long long row = blockIdx.x / csize;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  const int V = p.V;

  // Chunk c holds logits c N - shift .. + N - 1; the first and the last may be partly outside the row.
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int chunks = (int)(((long long)V + shift + N - 1) / N);
  const int c0 = (int)((long long)chunks * crank / csize), c1 = (int)((long long)chunks * (crank + 1) / csize);
  auto load = [&](int c) -> uint4 {
    const long long e = (long long)c * N - shift;
    if (e >= 0 && e + N <= V) return __ldcs(reinterpret_cast<const uint4*>(x + e));
    T v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = e + i >= 0 && e + i < V ? x[e + i] : T(-INFINITY);
    uint4 r;
    memcpy(&r, v, 16);
    return r;
  };
  const uint32_t low = sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u);
  const uint4 nothing = make_uint4(low, low, low, low);      // -inf

  uint4 next[INFLIGHT];
#pragma unroll
  for (int i = 0; i < INFLIGHT; ++i) {
    const int c = c0 + (int)threadIdx.x + i * THREADS;
    next[i] = c < c1 ? load(c) : nothing;
  }
  const long long id = p.ids[row];
  const bool valid = id >= 0 && id < V;
  const float xt = valid ? C::of(x[id]) : INFINITY;

  float m = -INFINITY, limit = -INFINITY;                    // reference (unset: -inf) and when to move it
  float2 S = make_float2(0.f, 0.f), W = S;
  float tm = -INFINITY;                                      // the thread's maximum and its first chunk
  int tc = c0 + (int)threadIdx.x, above = 0;
  const float2 L2 = make_float2(LOG2E, LOG2E);
  for (int c = c0 + (int)threadIdx.x; c < c1; c += INFLIGHT * THREADS) {
    uint4 now[INFLIGHT];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < INFLIGHT; ++i) {
      now[i] = next[i];
      const int cn = c + (INFLIGHT + i) * THREADS;
      next[i] = cn < c1 ? load(cn) : nothing;
    }
#pragma unroll
    for (int i = 0; i < INFLIGHT; ++i) {
      const float t = C::top(now[i]);
      top = max_nan(top, t);
      if (TOP && !(t <= tm) && tm == tm) tm = t, tc = c + i * THREADS;
    }
    if (top > limit) {
      if (m != -INFINITY) {
        const float t = fmaxf((m - top) * LOG2E, -160.f), f = exp2_approx(t);
        W = make_float2(fmaf(S.x, t, W.x) * f, fmaf(S.y, t, W.y) * f);
        S = make_float2(S.x * f, S.y * f);
      }
      m = top;
      limit = m + HEADROOM;
    }
    const float ref = m == -INFINITY ? 0.f : -m;
    const float2 r2 = make_float2(ref, ref);
    if constexpr (C::PACKED) {
      auto count = C::both(0.f);
      const auto t2 = C::both(xt);
#pragma unroll
      for (int i = 0; i < INFLIGHT; ++i)
#pragma unroll
        for (int j = 0; j < N / 2; ++j) count = __hadd2(count, __hgt2(C::pair(now[i], j), t2));   // exact: at most 16
      above += (int)(__low2float(count) + __high2float(count));
    } else {
#pragma unroll
      for (int i = 0; i < INFLIGHT; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) above += C::value(now[i], j) > xt;
    }
#pragma unroll
    for (int i = 0; i < INFLIGHT; ++i)
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        float2 y = mul2(add2(make_float2(C::value(now[i], j), C::value(now[i], j + 1)), r2), L2);
        y = make_float2(max_nan(y.x, -160.f), max_nan(y.y, -160.f));       // 2^-160 = 0 in fp32, 0 * -160 = 0
        const float2 e = make_float2(exp2_approx(y.x), exp2_approx(y.y));
        S = add2(S, e);
        W = fma2(e, y, W);
      }
  }

  // ---- the CTA's sums, relative to its largest reference ----
  float s = S.x + S.y, w = W.x + W.y;
  float bm = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) bm = fmaxf(bm, __shfl_xor_sync(~0u, bm, o));
  if (lane == 0) sh_m[warp] = bm;
  if (TOP) keys[threadIdx.x] = c0 + (int)threadIdx.x < c1 ? order_key(tm, (int)((long long)(tc + 1) * N - 1 - shift)) : 0;
  if (threadIdx.x == 0) n_list = n_cand = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WARPS; ++i) bm = fmaxf(bm, sh_m[i]);
  {
    const float t = m == -INFINITY ? 0.f : (m - bm) * LOG2E, f = exp2_approx(fmaxf(t, -160.f));
    w = f > 0.f ? fmaf(s, t, w) * f : 0.f;
    s = isnan(s) ? s : s * f;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s += __shfl_xor_sync(~0u, s, o);
    w += __shfl_xor_sync(~0u, w, o);
    above += __shfl_xor_sync(~0u, above, o);
  }
  if (lane == 0) sh_s[warp] = s, sh_w[warp] = w, sh_n[warp] = above;
  if (TOP && threadIdx.x < GROUPS) {
    unsigned long long g = 0;
#pragma unroll
    for (int i = 0; i < THREADS; i += GROUPS) g = max(g, keys[i + threadIdx.x]);
    group_key[threadIdx.x] = g;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float ts = 0.f, tw = 0.f;
    int tn = 0;
    for (int i = 0; i < WARPS; ++i) ts += sh_s[i], tw += sh_w[i], tn += sh_n[i];
    part.m = bm;
    part.s = ts;
    part.w = tw;
    part.above = tn;
    part.n_top = 0;
  }
  if constexpr (TOP) {
    const int k = p.top_k;
    // the k-th largest group maximum (0, below everything, where fewer than k groups hold anything)
    if (threadIdx.x < GROUPS) {
      const unsigned long long g = group_key[threadIdx.x];
      int r = 0;
      for (int i = 0; i < GROUPS; ++i) r += group_key[i] > g || (group_key[i] == g && i < (int)threadIdx.x);
      if (r == k - 1) bound_s = g;
    }
    __syncthreads();
    const unsigned long long bound = bound_s;
    if (keys[threadIdx.x] >= bound && c0 + (int)threadIdx.x < c1) list[atomicAdd(&n_list, 1)] = threadIdx.x;
    __syncthreads();
    const int per = (c1 - c0 + THREADS - 1) / THREADS, total = n_list * per;
    for (int i = threadIdx.x; i < total; i += THREADS) {
      const int c = c0 + list[i / per] + (i % per) * THREADS;
      if (c >= c1) continue;
      const uint4 v = load(c);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const long long e = (long long)c * N - shift + j;
        if (e >= 0 && e < V) {
          const unsigned long long key = order_key(C::value(v, j), (int)e);
          if (key >= bound) {
            const int at = atomicAdd(&n_cand, 1);
            if (at < CAND) cand[at] = key;
          }
        }
      }
    }
    __syncthreads();
    const int n = n_cand;
    if (n <= CAND) {
      for (int i = threadIdx.x; i < n; i += THREADS) {
        const unsigned long long mine = cand[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += cand[j] > mine;
        if (r < k) part.top[r] = mine;
      }
      if (threadIdx.x == 0) part.n_top = min(n, k);
    } else {
      // many large logits in few threads: one maximum of the whole slice after another
      unsigned long long last = ~0ull;
      for (int t = 0; t < k; ++t) {
        unsigned long long best = 0;
        for (int c = c0 + (int)threadIdx.x; c < c1; c += THREADS) {
          const uint4 v = load(c);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const long long e = (long long)c * N - shift + j;
            const unsigned long long key = e >= 0 && e < V ? order_key(C::value(v, j), (int)e) : 0;
            if (key < last) best = max(best, key);
          }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
        if (lane == 0) cand[warp] = best;
        __syncthreads();
        for (int i = 0; i < WARPS; ++i) best = max(best, cand[i]);
        __syncthreads();
        last = best;
        if (threadIdx.x == 0) part.top[t] = best;
      }
      if (threadIdx.x == 0) part.n_top = k;
    }
  }

  // ---- the cluster's parts, in the first CTA ----
  __syncthreads();
  if (csize > 1) cluster_sync_all();
  if (crank == 0) {
    const uint32_t mine = smem_u32(&part);
    auto word_of = [&](int q, uint32_t offset) {
      uint32_t v;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_rank(mine + offset, q)) : "memory");
      return v;
    };
    float M = -INFINITY, ts = 0.f, tw = 0.f;
    for (int q = 0; q < csize; ++q) M = fmaxf(M, __uint_as_float(word_of(q, offsetof(Part, m))));
    int tn = 0;
    for (int q = 0; q < csize; ++q) {
      const float qm = __uint_as_float(word_of(q, offsetof(Part, m))), qs = __uint_as_float(word_of(q, offsetof(Part, s))),
                  qw = __uint_as_float(word_of(q, offsetof(Part, w)));
      const float t = qm == -INFINITY ? 0.f : (qm - M) * LOG2E, f = exp2_approx(fmaxf(t, -160.f));
      tw += f > 0.f ? fmaf(qs, t, qw) * f : 0.f;
      ts += isnan(qs) ? qs : qs * f;
      tn += (int)word_of(q, offsetof(Part, above));
    }
    const RowResult r = logit_stat_finish(LogitStat{M, ts, tw * LN2}, xt, valid);
    if (threadIdx.x == 0) {
      p.logprob[row] = r.logprob;
      p.entropy[row] = r.entropy;
      p.lse[row] = r.lse;
      p.rank[row] = valid ? 1 + tn : 0;
    }
    if constexpr (TOP) {
      const float ls = logf(ts);
      auto write = [&](int at, unsigned long long key) {
        const int e = (int)~(uint32_t)key;
        const float f = C::of(x[e]);
        p.top_ids[row * p.top_k + at] = e;
        p.top_lp[row * p.top_k + at] = isnan(ts) ? NAN : M == -INFINITY ? -INFINITY : (f - M) - ls;
      };
      if (csize == 1) {
        for (int i = threadIdx.x; i < p.top_k; i += THREADS) write(i, part.top[i]);
      } else {
        int n = 0;
        for (int q = 0; q < csize; ++q) {
          const int nq = (int)word_of(q, offsetof(Part, n_top));
          for (int i = threadIdx.x; i < nq; i += THREADS) {
            const uint32_t at = offsetof(Part, top) + i * 8;
            cand[n + i] = (unsigned long long)word_of(q, at + 4) << 32 | word_of(q, at);
          }
          n += nq;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += THREADS) {
          const unsigned long long key = cand[i];
          int at = 0;
          for (int j = 0; j < n; ++j) at += cand[j] > key;
          if (at < p.top_k) write(at, key);
        }
      }
    }
  }
  if (csize > 1) cluster_sync_all();                         // the first CTA has read the others' shared memory
}

int num_sms() {
  constexpr int MAX_DEVICES = 64;
  static int cached[MAX_DEVICES] = {};
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return 148;
  if (cached[dev] <= 0)
    cached[dev] = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
  return cached[dev];
}

template <typename T, int THREADS>
int launch_t(const Args& p, int M, int cluster, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)M * cluster);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = p.top_k > 0 ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, THREADS, true>, p)
                                    : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, THREADS, false>, p);
  return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

template <typename T>
int launch(const Args& p, int M, cudaStream_t stream) {
  // CTAs of 128 threads for rows of up to 16 chunks a thread of those, where a large CTA would mostly synchronise.
  const long long chunks = (long long)p.V / Chunk<T>::N + 1;
  const bool small = chunks <= 2048;
  // As many CTAs a row as fill the SMs twice, each with two chunks a thread at least.
  const int threads = small ? 128 : 512;
  int cluster = 1;
  while (cluster < 8 && (long long)M * cluster < 2LL * num_sms() && chunks / (2 * cluster) >= 2 * threads) cluster *= 2;
  return small ? launch_t<T, 128>(p, M, cluster, stream) : launch_t<T, 512>(p, M, cluster, stream);
}

}  // namespace

extern "C" {

int b200_token_logprobs(const void* logits, int dtype, long long ld, int M, int V, const long long* ids, int top_k,
                        float* logprob, long long* rank, float* entropy, float* lse, long long* top_ids,
                        float* top_logprob, cudaStream_t stream) {
  if (M < 0) return -1;
  if (V < 1) return -2;
  if (ld < V) return -4;
  if (dtype < 0 || dtype > 2) return -5;
  if (top_k < 0 || top_k > MAX_TOP || top_k > V) return -6;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == 2 ? 3 : 1)) return -10;
  if (M == 0) return 0;
  if (M > (1 << 27)) return -1;                              // the grid's CTAs are counted in 32 bits
  const Args p{logits, ld, V, ids, top_k, logprob, rank, entropy, lse, top_ids, top_logprob};
  return dtype == 0 ? launch<__nv_bfloat16>(p, M, stream) : dtype == 1 ? launch<__half>(p, M, stream)
                                                                      : launch<float>(p, M, stream);
}

}  // extern "C"
