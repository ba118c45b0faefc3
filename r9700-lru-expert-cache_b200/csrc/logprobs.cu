// Log probabilities of given tokens from logits [M, V], with entropy, rank and top alternatives.
#include "score.cuh"

namespace {

using namespace b200;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// Order of (value, id) as one whole number: larger value first, then the lower id. NaN above +inf,
// -0 equal to +0.
__device__ __forceinline__ unsigned long long order_key(float x, int id) {
  uint32_t u = __float_as_uint(x + 0.f);
  u = isnan(x) ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (uint32_t)~id;
}

constexpr int THREADS = 512;

template <typename T>
__global__ void __launch_bounds__(THREADS)
    token_logprobs_kernel(const T* __restrict__ logits, long long ld, int V, const long long* __restrict__ ids,
                          int top_k, float* logprob, long long* rank, float* entropy, float* lse,
                          long long* top_ids, float* top_lp) {
  __shared__ LogitStat sh[THREADS / 32];
  __shared__ int sh_n[THREADS / 32];
  __shared__ unsigned long long sh_k[THREADS / 32];
  __shared__ float s_m, s_ls, s_s;
  const long long row = blockIdx.x;
  const T* x = logits + row * ld;
  const long long id = ids[row];
  const bool valid = id >= 0 && id < V;
  const float xt = valid ? to_f32(x[id]) : 0.f;
  LogitStat st = logit_stat_empty();
  int above = 0;
  for (int v = threadIdx.x; v < V; v += THREADS) {
    const float f = to_f32(x[v]);
    above += f > xt;
    LogitStat one = {f, f == -INFINITY ? 0.f : 1.f, 0.f};
    if (isnan(f) || f == INFINITY) one = LogitStat{0.f, NAN, NAN};
    st = logit_stat_merge(st, one);
  }
  for (int o = 16; o; o >>= 1) {
    LogitStat b = {__shfl_xor_sync(~0u, st.m, o), __shfl_xor_sync(~0u, st.s, o), __shfl_xor_sync(~0u, st.w, o)};
    st = logit_stat_merge(st, b);
    above += __shfl_xor_sync(~0u, above, o);
  }
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) sh[warp] = st, sh_n[warp] = above;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < THREADS / 32; ++i) st = logit_stat_merge(st, sh[i]), above += sh_n[i];
    const RowResult r = logit_stat_finish(st, xt, valid);
    logprob[row] = r.logprob;
    entropy[row] = r.entropy;
    lse[row] = r.lse;
    rank[row] = valid ? 1 + above : 0;
    s_m = st.m;
    s_s = st.s;
    s_ls = logf(st.s);
  }
  __syncthreads();
  unsigned long long last = ~0ull;
  for (int k = 0; k < top_k; ++k) {
    unsigned long long best = 0;
    for (int v = threadIdx.x; v < V; v += THREADS) {
      const unsigned long long key = order_key(to_f32(x[v]), v);
      if (key < last || k == 0) best = max(best, key);
    }
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
    if ((threadIdx.x & 31) == 0) sh_k[warp] = best;
    __syncthreads();
    for (int i = 0; i < THREADS / 32; ++i) best = max(best, sh_k[i]);
    __syncthreads();
    last = best;
    if (threadIdx.x == 0) {
      const int v = (int)~(uint32_t)best;
      const float f = to_f32(x[v]);
      top_ids[row * top_k + k] = v;
      top_lp[row * top_k + k] = isnan(s_s) ? NAN : s_m == -INFINITY ? -INFINITY : (f - s_m) - s_ls;
    }
  }
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
  if (top_k < 0 || top_k > 64 || top_k > V) return -6;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == 2 ? 3 : 1)) return -10;
  if (M == 0) return 0;
  if (dtype == 0)
    token_logprobs_kernel<<<M, THREADS, 0, stream>>>(static_cast<const __nv_bfloat16*>(logits), ld, V, ids, top_k,
                                                     logprob, rank, entropy, lse, top_ids, top_logprob);
  else if (dtype == 1)
    token_logprobs_kernel<<<M, THREADS, 0, stream>>>(static_cast<const __half*>(logits), ld, V, ids, top_k, logprob,
                                                     rank, entropy, lse, top_ids, top_logprob);
  else
    token_logprobs_kernel<<<M, THREADS, 0, stream>>>(static_cast<const float*>(logits), ld, V, ids, top_k, logprob,
                                                     rank, entropy, lse, top_ids, top_logprob);
  return (int)cudaGetLastError();
}

}  // extern "C"
