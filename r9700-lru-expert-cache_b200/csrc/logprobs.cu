// Log probabilities of given tokens from logits [M, V], with entropy, rank and top alternatives.
//
// One pass over a row. A thread walks 32-byte chunks of it (16 or 8 logits), keeping sums relative to a
// reference R, in units of log2 e, that it takes from the first logits it sees and moves only when one exceeds
// it by 6 (HEADROOM):
//   S = sum 2^y,  W = sum 2^y y,  y = x log2 e - R (one fused multiply-add),  and n = #{x > x_t};
// references differ between threads and meet at the end: moving a part to a larger R' is S 2^t and
// (W + S t) 2^t with t = R - R'. Then lse = (R + log2 S) ln 2, logprob = (x_t log2 e - R - log2 S) ln 2
// and entropy = (log2 S - W / S) ln 2. Their large terms cancel: y and W are held to 2^-24 of their sizes, so the
// headroom bounds the error, at about 6 2^-23. With 58 (4096 x 151936 with 20 alternatives 246 us for 248, 777 x 50001
// 25.8 for 26.3) a row whose one large logit stood 20 to 40 above the others had entropies off by 5e-6, in 512 rows
// 3e-5, and some below 0; with none, every larger logit a move, 259 and 27.3.
//
// The top alternatives cost the pass nothing but each thread's maximum and where it first was. The k-th
// largest of any k or more disjoint groups' maxima bounds the k-th largest logit from below, so only the
// few threads whose maximum reaches it can hold a top logit: their chunks are read again, and the handful
// of logits at or above the bound is ordered by counting. Order is (value descending, id ascending) as one
// 64-bit key, so nothing depends on timing.
//
// A row is shared by a cluster of 1 to 8 CTAs, so that few rows still occupy the SMs.
//
// What bounds it: without alternatives the row's bytes (4096 x 151936 bf16 in 205 us, 6.07 TB/s, 0.93 of a copy's
// rate), at about seven instructions a logit, close behind the issue slots. With 20 alternatives 248 us: the second
// reading, mostly from DRAM by then (27 KB of a row's 304), and seven barriers a row. Both in a burst of some
// milliseconds: at the power limit, whose clock settles near 1.63 GHz, 243 and 288. Few rows: latency, 4.7 us for
// one row, 8.4 with five alternatives. Rows with many logits equal to the bound are slow, since their chunks are all
// read for it and overflow into the last resort, a pass for each alternative: a mask that leaves fewer tokens than
// alternatives, or equal logits, took 14.6 ms at 4096 x 151936 with 20. Against this layout: one exponent by subtraction and multiplication and a
// clamp per logit on 16-byte chunks took 292 and 378 us; CTAs of 512 threads 227 and 294, of 128 threads 207 and 494.
#include <algorithm>

#include "score.cuh"
#include "tcgen05.cuh"

namespace {

using namespace b200;

constexpr int BIG = 256, MID = 128, SMALL = 64;   // threads of a CTA for long, ordinary and short rows
constexpr int MAX_TOP = 64;
constexpr int MAX_CLUSTER = 8;
constexpr int INFLIGHT = 2;                // chunks a thread loads at a time
constexpr float HEADROOM = 6.f;            // by which a logit may exceed its thread's reference, in units of log2 e
struct Raw {                               // 32 bytes of logits
  uint32_t w[8];
};

template <typename T>
struct Chunk;

template <>
struct Chunk<float> {
  static constexpr int N = 8;
  static constexpr bool PACKED = false;
  static constexpr uint32_t LOW = 0xff800000u;       // -inf
  __device__ static float value(const Raw& c, int i) { return __uint_as_float(c.w[i]); }
  __device__ static float top(const Raw& c) {
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = max_nan(value(c, i), value(c, i + 4));
    return max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3]));
  }
  __device__ static float of(float v) { return v; }
};

template <typename PairT>
__device__ __forceinline__ float top_of_pairs(const Raw& c) {
  auto pair = [&](int i) { return *reinterpret_cast<const PairT*>(&c.w[i]); };
  PairT m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = __hmax2_nan(pair(i), pair(i + 4));
  const PairT r = __hmax2_nan(__hmax2_nan(m[0], m[1]), __hmax2_nan(m[2], m[3]));
  return max_nan(__low2float(r), __high2float(r));
}

template <>
struct Chunk<__nv_bfloat16> {
  static constexpr int N = 16;
  static constexpr bool PACKED = true;
  static constexpr uint32_t LOW = 0xff80ff80u;
  using Pair = __nv_bfloat162;
  __device__ static Pair pair(const Raw& c, int i) { return *reinterpret_cast<const Pair*>(&c.w[i]); }
  __device__ static float value(const Raw& c, int i) {
    return __uint_as_float(i & 1 ? c.w[i >> 1] & 0xffff0000u : c.w[i >> 1] << 16);
  }
  __device__ static float top(const Raw& c) { return top_of_pairs<Pair>(c); }
  __device__ static float of(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static Pair both(float v) { return __float2bfloat162_rn(v); }
};

template <>
struct Chunk<__half> {
  static constexpr int N = 16;
  static constexpr bool PACKED = true;
  static constexpr uint32_t LOW = 0xfc00fc00u;
  using Pair = __half2;
  __device__ static Pair pair(const Raw& c, int i) { return *reinterpret_cast<const Pair*>(&c.w[i]); }
  __device__ static float value(const Raw& c, int i) {
    return i & 1 ? __high2float(pair(c, i >> 1)) : __low2float(pair(c, i >> 1));
  }
  __device__ static float top(const Raw& c) { return top_of_pairs<Pair>(c); }
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

__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);       // (NaN's key gives a NaN)
}

// 32 aligned bytes, read once.
__device__ __forceinline__ Raw ld_stream(const void* p) {
  Raw r;
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                 "=r"(r.w[7])
               : "l"(p));
  return r;
}

// Sums relative to `from` made relative to `to` >= from. A part without logits above -inf has no reference.
__device__ __forceinline__ void move_to(float from, float to, float& s, float& w) {
  const float t = from == -INFINITY ? 0.f : fmaxf(from - to, LOWEST_Y), f = exp2_approx(t);
  w = f > 0.f ? fmaf(s, t, w) * f : 0.f;
  s = isnan(s) ? s : s * f;
}

// What a CTA of a row's cluster leaves in the first one's shared memory.
struct Part {
  float ref, s, w;
  int above, any;                          // any: a logit above -inf
  int pad;
  unsigned long long top[MAX_TOP];         // its top_k keys, 0 where it has fewer logits
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
  // Chunks and logits at or above the bound that are kept; more take the slow way.
  constexpr int HITS = THREADS, CAND = 4 * THREADS;
  __shared__ Part parts[MAX_CLUSTER];
  __shared__ float sh_m[WARPS], sh_s[WARPS], sh_w[WARPS];
  __shared__ int sh_n[WARPS];
  __shared__ unsigned long long keys[TOP ? THREADS : 1], group_key[TOP ? MAX_TOP : 1], cand[TOP ? CAND : 1];
  __shared__ unsigned long long own_top[TOP ? MAX_TOP : 1];
  __shared__ int list[TOP ? THREADS : 1], hits[TOP ? HITS : 1];
  __shared__ Raw hit_chunk[TOP ? HITS : 1];
  __shared__ int n_list, n_hits, n_cand;
  __shared__ unsigned long long bound_s;
  const int crank = (int)cluster_rank(), csize = (int)cluster_size();
  const long long row = blockIdx.x / csize;
  if (csize > 1) cluster_arrive();                           // (waited for before the first store to another CTA)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  const int V = p.V;

  // Chunk c holds logits c N - shift .. + N - 1; the first and the last may be partly outside the row.
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 31) / sizeof(T));
  const int chunks = (int)(((long long)V + shift + N - 1) / N);
  const int c0 = (int)((long long)chunks * crank / csize), c1 = (int)((long long)chunks * (crank + 1) / csize);
  const char* aligned_row = reinterpret_cast<const char*>(x - shift);
  auto guarded = [&](int c) {
    Raw r;
    const long long e = (long long)c * N - shift;
    if (c < c1 && e >= 0 && e + N <= V) return ld_stream(aligned_row + (long long)c * 32);
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = C::LOW;
    if (c < c1) {
      T v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = e + i >= 0 && e + i < V ? x[e + i] : T(-INFINITY);
      memcpy(&r, v, 32);
    }
    return r;
  };
  // Passes of INFLIGHT chunks a thread, contiguous over the CTA; pass q is whole if no chunk of it needs a guard.
  constexpr int PASS = INFLIGHT * THREADS;
  const int mine = c0 + (int)threadIdx.x, passes = (c1 - c0 + PASS - 1) / PASS;
  const int whole0 = shift != 0 && crank == 0 ? 1 : 0;
  const int whole1 = (c1 - c0 - (crank == csize - 1 && (V + shift) % N != 0 ? 1 : 0)) / PASS;
  auto load_pass = [&](int q, Raw (&to)[INFLIGHT]) {
    const int c = mine + q * PASS;
    if (q >= whole0 && q < whole1) {
      const char* at = aligned_row + (long long)c * 32;
#pragma unroll
      for (int i = 0; i < INFLIGHT; ++i) to[i] = ld_stream(at + i * THREADS * 32);
    } else {
#pragma unroll
      for (int i = 0; i < INFLIGHT; ++i) to[i] = guarded(c + i * THREADS);
    }
  };

  Raw next[INFLIGHT];
  load_pass(0, next);
  const long long id = p.ids[row];
  const bool valid = id >= 0 && id < V;
  const float xt = valid ? C::of(x[id]) : INFINITY;

  float ref = -INFINITY, limit = -LARGE;                     // reference (unset: -inf) and the logit that moves it
  bool some = false;                                         // a logit above -inf
  float2 S = make_float2(0.f, 0.f), W = S;
  float tm = -INFINITY;                                      // the thread's maximum and its first chunk
  int tc = mine, above = 0;
  const float2 L2 = make_float2(LOG2E, LOG2E);
  for (int q = 0; q < passes; ++q) {
    Raw now[INFLIGHT];
#pragma unroll
    for (int i = 0; i < INFLIGHT; ++i) now[i] = next[i];
    if (q + 1 < passes) load_pass(q + 1, next);
#pragma unroll
    for (int i = 0; i < INFLIGHT; ++i) {
      const int c = mine + q * PASS + i * THREADS;
      if (q >= whole1 && c >= c1) break;                     // (whole warps leave the last pass here)
      const float top = C::top(now[i]);
      if (TOP && !(top <= tm) && tm == tm) tm = top, tc = c;
      some |= top > -INFINITY;
      if (top > limit) {
        const float moved = top * LOG2E;
        if (ref != -INFINITY) {
          const float t = fmaxf(ref - moved, LOWEST_Y), f = exp2_approx(t);
          W = make_float2(fmaf(S.x, t, W.x) * f, fmaf(S.y, t, W.y) * f);
          S = make_float2(S.x * f, S.y * f);
        }
        ref = moved;
        limit = top + HEADROOM / LOG2E;
      }
      if (!(top <= xt)) {                                    // (top is NaN where the chunk holds one: its others count)
        if constexpr (C::PACKED) {
          auto count = C::both(0.f);
          const auto t2 = C::both(xt);
#pragma unroll
          for (int j = 0; j < N / 2; ++j) count = __hadd2(count, __hgt2(C::pair(now[i], j), t2));   // exact: at most 8
          above += (int)(__low2float(count) + __high2float(count));
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j) above += C::value(now[i], j) > xt;
        }
      }
      const float r = ref == -INFINITY ? 0.f : -ref;
      const float2 r2 = make_float2(r, r);
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        float2 y = fma2(make_float2(C::value(now[i], j), C::value(now[i], j + 1)), L2, r2);
        y = make_float2(max_nan(y.x, LOWEST_Y), max_nan(y.y, LOWEST_Y));
        const float2 e = make_float2(exp2_approx(y.x), exp2_approx(y.y));
        S = add2(S, e);
        W = fma2(e, y, W);
      }
    }
  }

  // ---- the CTA's sums, relative to its largest reference ----
  float s = S.x + S.y, w = W.x + W.y;
  float bref = ref;
#pragma unroll
  for (int o = 16; o; o >>= 1) bref = fmaxf(bref, __shfl_xor_sync(~0u, bref, o));
  if (lane == 0) sh_m[warp] = bref;
  if (TOP) keys[threadIdx.x] = mine < c1 ? order_key(tm, (int)((long long)(tc + 1) * N - 1 - shift)) : 0;
  if (threadIdx.x == 0) n_list = n_hits = n_cand = 0;
  if (TOP && threadIdx.x < MAX_TOP) own_top[threadIdx.x] = 0;
  // Groups: threads of equal number modulo 32, or 64 where 32 would bound many alternatives loosely.
  const int groups = p.top_k > 16 ? 64 : 32;
  const int any = __syncthreads_or(some);
#pragma unroll
  for (int i = 0; i < WARPS; ++i) bref = fmaxf(bref, sh_m[i]);
  move_to(ref, bref, s, w);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s += __shfl_xor_sync(~0u, s, o);
    w += __shfl_xor_sync(~0u, w, o);
    above += __shfl_xor_sync(~0u, above, o);
  }
  if (lane == 0) sh_s[warp] = s, sh_w[warp] = w, sh_n[warp] = above;
  if (TOP && (int)threadIdx.x < groups) {
    unsigned long long g = 0;
    for (int i = threadIdx.x; i < THREADS; i += groups) g = max(g, keys[i]);
    group_key[threadIdx.x] = g;
  }
  __syncthreads();
  if constexpr (TOP) {
    const int k = p.top_k;
    // the k-th largest group maximum (0, below everything, where fewer than k groups hold anything)
    if ((int)threadIdx.x < groups) {
      const unsigned long long g = group_key[threadIdx.x];
      int r = 0;
#pragma unroll 16
      for (int i = 0; i < groups; ++i) r += group_key[i] > g || (group_key[i] == g && i < (int)threadIdx.x);
      if (r == k - 1) bound_s = g;
    }
    __syncthreads();
    const unsigned long long bound = bound_s;
    if (keys[threadIdx.x] >= bound && mine < c1) list[atomicAdd(&n_list, 1)] = threadIdx.x;
    __syncthreads();
    const int per = (c1 - c0 + THREADS - 1) / THREADS, total = n_list * per;
    constexpr int AGAIN = 3;                                 // chunks read again at a time
    for (int i0 = threadIdx.x; i0 < total; i0 += AGAIN * THREADS) {
      Raw v[AGAIN];
      int at[AGAIN];
#pragma unroll
      for (int a = 0; a < AGAIN; ++a) {
        const int i = i0 + a * THREADS;
        at[a] = i < total ? c0 + list[i / per] + (i % per) * THREADS : c1;
        v[a] = guarded(at[a]);
      }
#pragma unroll
      for (int a = 0; a < AGAIN; ++a)
        if (at[a] < c1 && order_key(C::top(v[a]), 0) >= (bound & 0xffffffff00000000ull)) {
          const int put = atomicAdd(&n_hits, 1);
          if (put < HITS) hits[put] = at[a], hit_chunk[put] = v[a];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(n_hits, HITS) * N; i += THREADS) {
      const long long e = (long long)hits[i / N] * N - shift + i % N;
      const float f = C::of(reinterpret_cast<const T*>(hit_chunk)[i]);
      const unsigned long long key = e >= 0 && e < V ? order_key(f, (int)e) : 0;
      if (key >= bound && key != 0) {
        const int put = atomicAdd(&n_cand, 1);
        if (put < CAND) cand[put] = key;
      }
    }
    __syncthreads();
    const int n = n_cand;
    if (n <= CAND && n_hits <= HITS) {
      for (int i = threadIdx.x; i < n; i += THREADS) {
        const unsigned long long key = cand[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += cand[j] > key;
        if (r < k) own_top[r] = key;
      }
    } else {
      // many large logits in few threads: one maximum of the whole slice after another
      unsigned long long last = ~0ull;
      for (int t = 0; t < k; ++t) {
        unsigned long long best = 0;
        for (int c = mine; c < c1; c += THREADS) {
          const Raw v = guarded(c);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const long long e = (long long)c * N - shift + j;
            const unsigned long long key = e >= 0 && e < V ? order_key(C::value(v, j), (int)e) : 0;
            if (t == 0 || key < last) best = max(best, key);    // (NaN at id 0 has the largest key there is)
          }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
        if (lane == 0) cand[warp] = best;
        __syncthreads();
        for (int i = 0; i < WARPS; ++i) best = max(best, cand[i]);
        __syncthreads();
        last = best;
        if (threadIdx.x == 0) own_top[t] = best;
      }
    }
  }

  // ---- the cluster's parts, in the first CTA ----
  __syncthreads();
  if (csize > 1) cluster_wait();                             // the first CTA has started
  {
    const uint32_t to = map_to_rank(smem_u32(&parts[crank]), 0);
    if (threadIdx.x == 0) {
      float ts = 0.f, tw = 0.f;
      int tn = 0;
      for (int i = 0; i < WARPS; ++i) ts += sh_s[i], tw += sh_w[i], tn += sh_n[i];
      st_cluster(to + offsetof(Part, ref), __float_as_uint(bref));
      st_cluster(to + offsetof(Part, s), __float_as_uint(ts));
      st_cluster(to + offsetof(Part, w), __float_as_uint(tw));
      st_cluster(to + offsetof(Part, above), (uint32_t)tn);
      st_cluster(to + offsetof(Part, any), (uint32_t)any);
    }
    if (TOP && (int)threadIdx.x < p.top_k) {
      const unsigned long long key = own_top[threadIdx.x];
      const uint32_t at = to + offsetof(Part, top) + threadIdx.x * 8;
      st_cluster(at, (uint32_t)key);
      st_cluster(at + 4, (uint32_t)(key >> 32));
    }
  }
  if (csize > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (crank == 0) {
    float R = -INFINITY, ts = 0.f, tw = 0.f;
    for (int q = 0; q < csize; ++q) R = fmaxf(R, parts[q].ref);
    int tn = 0, found = 0;
    for (int q = 0; q < csize; ++q) {
      float qs = parts[q].s, qw = parts[q].w;
      move_to(parts[q].ref, R, qs, qw);
      ts += qs;
      tw += qw;
      tn += parts[q].above;
      found |= parts[q].any;
    }
    const bool huge = found && !(fabsf(R) < LARGE * LOG2E);
    const bool nan = !huge && isnan(ts), empty = !found && !nan;
    LogitStat st = logit_stat_empty();
    if (huge) {
      for (int e = threadIdx.x; e < V; e += THREADS) {
        const float f = C::of(x[e]);
        if (!(f < INFINITY)) st = LogitStat{0.f, NAN, NAN};
        if (f > -INFINITY) st = logit_stat_merge(st, LogitStat{f, 1.f, 0.f});
      }
#pragma unroll
      for (int o = 16; o; o >>= 1)
        st = logit_stat_merge(st, LogitStat{__shfl_xor_sync(~0u, st.m, o), __shfl_xor_sync(~0u, st.s, o),
                                            __shfl_xor_sync(~0u, st.w, o)});
      __syncthreads();
      if (lane == 0) sh_m[warp] = st.m, sh_s[warp] = st.s, sh_w[warp] = st.w;
      __syncthreads();
      st = logit_stat_empty();
      for (int i = 0; i < WARPS; ++i) st = logit_stat_merge(st, LogitStat{sh_m[i], sh_s[i], sh_w[i]});
    }
    const float ls = log2f(ts), lse = (R + ls) * LN2;
    auto logprob = [&](float v) -> float {
      if (nan) return NAN;
      if (empty) return -INFINITY;
      if (huge) return logit_stat_finish(st, v, true).logprob;
      if (v < -1e38f) return v - lse;                        // (v log2 e may be below fp32's range)
      return fminf((fmaf(v, LOG2E, -R) - ls) * LN2, 0.f);
    };
    if (threadIdx.x == 0) {
      const RowResult h = logit_stat_finish(st, xt, valid);
      p.logprob[row] = valid ? logprob(xt) : NAN;
      p.entropy[row] = nan ? NAN : empty ? 0.f : huge ? h.entropy : fmaxf(ls - tw / ts, 0.f) * LN2;
      p.lse[row] = nan ? NAN : empty ? -INFINITY : huge ? h.lse : lse;
      p.rank[row] = valid ? 1 + tn : 0;
    }
    if constexpr (TOP) {
      auto write = [&](int at, unsigned long long key) {
        p.top_ids[row * p.top_k + at] = (int)~(uint32_t)key;
        p.top_lp[row * p.top_k + at] = logprob(key_value(key));
      };
      const int k = p.top_k;
      if (csize == 1) {
        for (int i = threadIdx.x; i < k; i += THREADS) write(i, parts[0].top[i]);
      } else {
        for (int i = threadIdx.x; i < csize * k; i += THREADS) {
          const unsigned long long key = parts[i / k].top[i % k];
          int at = key == 0 ? k : 0;
          for (int q = 0; q < csize; ++q)
            for (int j = 0; j < k; ++j) at += parts[q].top[j] > key;
          if (at < k) write(at, key);
        }
      }
    }
  }
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
  // CTAs of few threads for short rows, which mostly synchronise: up to 1024 chunks, and with many rows up to 4096
  // (777 x 50001 f16 with 8 alternatives 26.5 us in 128 threads and 28.0 in 256, 2000 x 20000 bf16 30.2 and 36.4, but
  // 16 x 32000 9.1 and 8.2, and 4096 x 151936 with 20 alternatives 494 and 258: a top logit's thread has more chunks
  // to read again. One warp a row took 142 us for 32 at 4096 x 2000 with 20.)
  const long long chunks = (long long)p.V / Chunk<T>::N + 1;
  const int threads = chunks <= 1024 ? SMALL : chunks <= 4096 && M >= num_sms() ? MID : BIG;
  // CTAs a row, each with two chunks a thread at least: the fewest turns of the SMs' CTAs, a turn being a CTA's
  // share of the row at its share of the bandwidth and about 8 us of reduction.
  const long long slots = (long long)(1024 / threads) * num_sms();
  const double row_us = (double)p.V * sizeof(T) * slots / 5.9e6;
  int cluster = 1;
  double best = 1e300;
  for (int c = 1; c <= MAX_CLUSTER && (c == 1 || chunks / c >= 2 * threads); c *= 2) {
    const double us = (double)((M * (long long)c + slots - 1) / slots) * (row_us / c + 8.);
    if (us < best) best = us, cluster = c;
  }
  return threads == SMALL ? launch_t<T, SMALL>(p, M, cluster, stream)
                          : threads == MID ? launch_t<T, MID>(p, M, cluster, stream)
                                           : launch_t<T, BIG>(p, M, cluster, stream);
}

}  // namespace

extern "C" {

int b200_token_logprobs(const void* logits, int dtype, long long ld, int M, int V, const long long* ids, int top_k,
                        float* logprob, long long* rank, float* entropy, float* lse, long long* top_ids,
                        float* top_logprob, cudaStream_t stream) {
  if (M < 0 || M > (1 << 27)) return -1;                     // (a grid's CTAs and a row's chunks are counted in 32 bits)
  if (V < 1 || V > (1 << 30)) return -2;
  if (ld < V) return -4;
  if (dtype < 0 || dtype > 2) return -5;
  if (top_k < 0 || top_k > MAX_TOP || top_k > V) return -6;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == 2 ? 3 : 1)) return -10;
  if (M == 0) return 0;
  const Args p{logits, ld, V, ids, top_k, logprob, rank, entropy, lse, top_ids, top_logprob};
  return dtype == 0 ? launch<__nv_bfloat16>(p, M, stream) : dtype == 1 ? launch<__half>(p, M, stream)
                                                                      : launch<float>(p, M, stream);
}

}  // extern "C"
