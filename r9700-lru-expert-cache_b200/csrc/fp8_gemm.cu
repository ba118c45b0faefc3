// FP8 128x128 block-scaled matrix product for any number of tokens, and the same product reduced
// to the log probabilities of given tokens.
#include "score.cuh"

namespace {

using namespace b200;

__device__ int g_score_err = 0;

struct Operands {
  const uint8_t* x;
  long long ldx;
  const float* xs;
  long long xs_row, xs_col;
  const uint8_t* w;
  long long ldw;
  int packed;
  const float* ws;
  long long ws_row;
  int M, N, K;
};

// Byte of weight element (n, k): row-major, or the strip pack [N/16][K/128][16 rows][128 B] with
// 16-byte chunk c of strip row r at chunk c ^ (r & 7).
__device__ __forceinline__ long long weight_at(const Operands& p, int n, int k) {
  if (!p.packed) return n * p.ldw + k;
  const int r = n & 15, c = (k & 127) >> 4;
  return ((long long)(n >> 4) * (p.K >> 7) + (k >> 7)) * 2048 + r * 128 + ((c ^ (r & 7)) << 4) + (k & 15);
}

__device__ __forceinline__ float e4m3_to_f32(uint8_t b) {
  __nv_fp8_e4m3 v;
  v.__x = b;
  return float(v);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

constexpr int T = 64;

// One 64 x 64 tile of y per CTA, 256 threads of 4 x 4 outputs, K in steps of 16.
__device__ __forceinline__ void product_tile(const Operands& p, int m0, int n0, float (&acc)[4][4]) {
  __shared__ float xa[16][T + 1], wa[16][T + 1];
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  float part[4][4] = {};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  for (int k0 = 0; k0 < p.K; k0 += 16) {
    for (int e = threadIdx.x; e < 16 * T; e += 256) {
      const int r = e >> 4, k = e & 15;
      xa[k][r] = m0 + r < p.M ? e4m3_to_f32(p.x[(m0 + r) * p.ldx + k0 + k]) : 0.f;
      wa[k][r] = n0 + r < p.N ? e4m3_to_f32(p.w[weight_at(p, n0 + r, k0 + k)]) : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < 16; ++k)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) part[i][j] = fmaf(xa[k][ty * 4 + i], wa[k][tx * 4 + j], part[i][j]);
    __syncthreads();
    if ((k0 & 127) == 112 || k0 + 16 >= p.K) {
      const int b = k0 >> 7;
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
          const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
          const float s = m < p.M && n < p.N ? p.xs[m * p.xs_row + b * p.xs_col] * p.ws[(n >> 7) * p.ws_row + b] : 0.f;
          acc[i][j] = fmaf(part[i][j], s, acc[i][j]);
          part[i][j] = 0.f;
        }
    }
  }
}

template <typename OUT>
__global__ void __launch_bounds__(256) gemm_kernel(Operands p, OUT* y, long long ldy) {
  float acc[4][4];
  const int m0 = blockIdx.y * T, n0 = blockIdx.x * T;
  product_tile(p, m0, n0, acc);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + (threadIdx.x >> 4) * 4 + i, n = n0 + (threadIdx.x & 15) * 4 + j;
      if (m < p.M && n < p.N) y[m * ldy + n] = from_f32<OUT>(acc[i][j]);
    }
}

// part [column tile][3][M]; token [M]
__global__ void __launch_bounds__(256)
    head_kernel(Operands p, const long long* __restrict__ ids, float* __restrict__ part, float* __restrict__ token) {
  __shared__ float tile[T][T + 1];
  float acc[4][4];
  const int m0 = blockIdx.y * T, n0 = blockIdx.x * T;
  product_tile(p, m0, n0, acc);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) tile[(threadIdx.x >> 4) * 4 + i][(threadIdx.x & 15) * 4 + j] = acc[i][j];
  __syncthreads();
  const int m = m0 + threadIdx.x;
  if (threadIdx.x < T && m < p.M) {
    LogitStat st = logit_stat_empty();
    const long long id = ids[m];
    for (int j = 0; j < T && n0 + j < p.N; ++j) {
      const float f = tile[threadIdx.x][j];
      if (n0 + j == id) token[m] = f;
      LogitStat one = {f, f == -INFINITY ? 0.f : 1.f, 0.f};
      if (isnan(f) || f == INFINITY) one = LogitStat{0.f, NAN, NAN};
      st = logit_stat_merge(st, one);
    }
    float* o = part + (long long)blockIdx.x * 3 * p.M + m;
    o[0] = st.m;
    o[p.M] = st.s;
    o[2LL * p.M] = st.w;
  }
}

__global__ void __launch_bounds__(128)
    head_merge_kernel(const float* __restrict__ part, const float* __restrict__ token,
                      const long long* __restrict__ ids, int tiles, int M, int N, float* logprob, float* entropy,
                      float* lse) {
  const int m = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (m >= M) return;
  LogitStat st = logit_stat_empty();
  for (int t = threadIdx.x & 31; t < tiles; t += 32) {
    const float* o = part + (long long)t * 3 * M + m;
    st = logit_stat_merge(st, LogitStat{o[0], o[M], o[2LL * M]});
  }
  for (int o = 16; o; o >>= 1)
    st = logit_stat_merge(st, LogitStat{__shfl_xor_sync(~0u, st.m, o), __shfl_xor_sync(~0u, st.s, o),
                                        __shfl_xor_sync(~0u, st.w, o)});
  if ((threadIdx.x & 31) == 0) {
    const bool valid = ids[m] >= 0 && ids[m] < N;
    const RowResult r = logit_stat_finish(st, valid ? token[m] : 0.f, valid);
    logprob[m] = r.logprob;
    entropy[m] = r.entropy;
    lse[m] = r.lse;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_operands(const Operands& p) {
  if (p.M < 0) return -1;
  if (p.N < 1 || (p.packed && p.N % 16)) return -2;
  if (p.K < 16 || p.K % 16 || (p.packed && p.K % 128)) return -3;
  if (p.ldx < p.K || p.ldx % 16 || (!p.packed && (p.ldw < p.K || p.ldw % 16))) return -4;
  if (!aligned16(p.x) || !aligned16(p.w)) return -10;
  return 0;
}

int column_tiles(int N) { return (N + T - 1) / T; }

}  // namespace

extern "C" {

int b200_fp8_block_gemm(const void* qx, long long ldx, const float* xs, long long xs_row, long long xs_col,
                        const void* wq, long long ldw, int packed, const float* ws, long long ws_row, void* y,
                        long long ldy, int y_dtype, int M, int N, int K, cudaStream_t stream) {
  const Operands p{static_cast<const uint8_t*>(qx), ldx, xs, xs_row, xs_col, static_cast<const uint8_t*>(wq), ldw,
                   packed, ws, ws_row, M, N, K};
  const int rc = check_operands(p);
  if (rc != 0) return rc;
  if (ldy < N) return -4;
  if (y_dtype < 0 || y_dtype > 2) return -5;
  if (reinterpret_cast<uintptr_t>(y) & (y_dtype == 2 ? 3 : 1)) return -10;
  if (M == 0) return 0;
  const dim3 grid(column_tiles(N), (M + T - 1) / T);
  if (y_dtype == 0)
    gemm_kernel<<<grid, 256, 0, stream>>>(p, static_cast<__nv_bfloat16*>(y), ldy);
  else if (y_dtype == 1)
    gemm_kernel<<<grid, 256, 0, stream>>>(p, static_cast<__half*>(y), ldy);
  else
    gemm_kernel<<<grid, 256, 0, stream>>>(p, static_cast<float*>(y), ldy);
  return (int)cudaGetLastError();
}

long long b200_fp8_head_logprobs_workspace_bytes(int M, int N) {
  if (M <= 0 || N <= 0) return 0;
  return (3LL * column_tiles(N) + 1) * M * 4;
}

int b200_fp8_head_logprobs(const void* qx, long long ldx, const float* xs, long long xs_row, long long xs_col,
                           const void* wq, long long ldw, int packed, const float* ws, long long ws_row,
                           const long long* ids, int M, int N, int K, float* logprob, float* entropy, float* lse,
                           void* workspace, long long workspace_bytes, cudaStream_t stream) {
  const Operands p{static_cast<const uint8_t*>(qx), ldx, xs, xs_row, xs_col, static_cast<const uint8_t*>(wq), ldw,
                   packed, ws, ws_row, M, N, K};
  const int rc = check_operands(p);
  if (rc != 0) return rc;
  if (M == 0) return 0;
  if (workspace == nullptr || workspace_bytes < b200_fp8_head_logprobs_workspace_bytes(M, N)) return -9;
  if (!aligned16(workspace)) return -10;
  float* token = static_cast<float*>(workspace);
  float* part = token + M;
  head_kernel<<<dim3(column_tiles(N), (M + T - 1) / T), 256, 0, stream>>>(p, ids, part, token);
  head_merge_kernel<<<(M + 3) / 4, 128, 0, stream>>>(part, token, ids, column_tiles(N), M, N, logprob, entropy, lse);
  return (int)cudaGetLastError();
}

int b200_score_error(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_score_err, sizeof(int)) != cudaSuccess) return -1;
  if (reset) {
    const int z = 0;
    if (cudaMemcpyToSymbol(g_score_err, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

}  // extern "C"
