// FP8 128x128 block-scaled matrix product for any number of tokens, and the same product reduced
// to the log probabilities of given tokens.
//
//   y[m, n] = sum_b xs[m, b] ws[n / 128, b] D_b[m, n],   D_b[m, n] = sum_{k in block b} qx[m, k] wq[n, k]
//
// Each D_b is one accumulator of the tensor core (fp32, TMEM): 128 tokens x BN weight rows, 128 K. The
// weight's scale is one number over 128 rows and the token's is one number per TMEM lane, so a thread that
// holds a lane's columns needs one factor per block of 128 columns: the promotion of D_b into the running sum is
// a tcgen05.ld and one fused multiply-add per value, in registers, while the MMAs fill the other accumulators.
//   warp 0     one lane copies the tiles (tensor maps: zeros beyond M, N and K) into a ring of stages;
//   warps 1, 3 one lane each issues MMAs, four of K = 32 a 128-K block, into a fresh accumulator;
//   warp 2     puts the factors xs ws of four 128-K blocks at a time into shared memory (each promoting thread
//              reading its own row's scales cost more L1 wavefronts than the block's MMAs take);
//   warps 4-11 two groups of four, each with half of the columns: promote, then write the tile.
// CTAs (or pairs) walk the tiles, rows first within groups of row tiles, so that tiles in flight share weights.
//
// Above 128 rows two CTAs share a tile of 256 rows x 256 columns (cta_group::2): a stage is 32 KB a CTA instead of
// 48, which the L2 and the shared memory feel (8192 x 10240 x 2560 201 us, one CTA 216). What bounds it: at a fixed
// number of tiles and K from 512 to 10240 a block takes 830 to 870 clocks, 512 of them its MMAs (the tensor pipe is
// active 59 % of the time), and a tile 2400 more. DRAM (11 %), L2 (34 %) and issue slots (48 %) are not full; which
// part of an accumulator's way from commit through two waits (110 to 160 clocks each), eight TMEM loads with their 64
// multiply-adds and release to the issuing CTA makes the difference has not been told apart. A tile of the head costs
// about 7000 clocks beside its blocks, statistics that the MMAs do not hide. And the power limit: the product takes 200
// to 209 us in a burst of some milliseconds (up to 2150 TFLOP/s), 240 once the clock has settled, at 1470 MHz. Few
// tokens stream the weight: 8 x 151936 x 2560 takes 67 us, 5.8 TB/s.
#include <algorithm>
#include <cstdlib>

#include <cudaTypedefs.h>

#include "score.cuh"
#include "tcgen05.cuh"

namespace {

using namespace b200;

__device__ int g_score_err = 0;

constexpr int EPI_GROUPS = 2, EPI_WARPS = 4 * EPI_GROUPS;
constexpr int THREADS = 32 * (4 + EPI_WARPS);
constexpr int BM = 128;                    // token rows of a CTA's tile (TMEM lanes)
constexpr int SMEM_CAP = 227 * 1024;
constexpr int OUT_BUFS = 2, OUT_BUF = 4096; // a warp's output buffers: bf16 and f16 tiles fit whole
constexpr int MAX_STAGES = 12;
// Every CTA takes all of TMEM, so no two may share an SM (a second one's allocation would wait, and CTAs of
// two clusters could wait for each other): each asks for more than half of the shared memory.
constexpr int SMEM_MIN = 116 * 1024;
constexpr int FGROUP = 4;                  // 128-K blocks whose factors are written at a time
constexpr int F_LD = 2 * BM + 8;           // of one block: [column block][row], padded against bank conflicts
constexpr int GROUP_ROWS = 16;             // row tiles that share a stretch of the weight

struct Product {
  const float* xs;
  long long xs_row, xs_col;
  const float* ws;
  long long ws_row;
  int M, N, K;
  int packed;
  int box_m;                               // token rows that a stage's copy brings
  int row_tiles, col_tiles;
  int nstage;
  int quarters, a_bytes;                   // quarters of 32 rows with tokens; bytes of a stage's token rows (CG = 1)
  // product
  void* y;
  long long ldy;
  int tma_out;                             // y's base and rows are 16-byte aligned
  uint32_t tries;                          // of a pipeline wait before it gives up
  // head: of every row and column tile {m, s, w, 0}; of every row its token's logit
  const long long* ids;
  float4* part;
  float* token;
};
static_assert(sizeof(Product) <= 128, "one word more and the 256-column tiles spill 120 bytes a thread");

enum Out { OUT_BF16 = 0, OUT_F16 = 1, OUT_F32 = 2, OUT_STATS = 3 };

// How a tile's 128-K block goes through TMEM. BN <= 128: one accumulator of BN columns, half of it for each
// epilogue group. BN = 256: two accumulators of 128 columns, one for each group, with barriers of their own, so
// that four are in flight: an accumulator's way from its last MMA through commit, load and release back to its
// next MMA takes longer than the other one's MMAs.
template <int BN>
struct Tile {
  static constexpr int UNITS = BN == 256 ? 2 : 1;   // accumulators of a 128-K block
  static constexpr int UN = BN / UNITS;             // their columns
  static constexpr int W = BN / EPI_GROUPS;         // columns of one epilogue group
  static constexpr int NBUF = 512 / UN > 8 ? 8 : 512 / UN;
  static constexpr int RELEASERS = UNITS == 2 ? EPI_WARPS / 2 : EPI_WARPS;   // warps of a CTA that read one
  static constexpr int BLOCKS = BN > 128 ? BN / 128 : 1;   // weight scales of a tile's 128-K block
  // Register split of the launch's 168 registers a thread: the running sums of BN = 256 need more.
  static constexpr bool SPLIT_REGS = BN == 256;
  static constexpr int LAUNCH_REGS = 168, EPI_REGS = 216, OTHER_REGS = 72;
  static_assert(EPI_REGS * EPI_WARPS + OTHER_REGS * 4 <= LAUNCH_REGS * (EPI_WARPS + 4), "more than the launch brings");
};

// Tile number -> (row tile, column tile).
__device__ __forceinline__ void tile_at(const Product& p, int t, int& rt, int& ct) {
  const int per_group = GROUP_ROWS * p.col_tiles, g = t / per_group, r = t - g * per_group;
  const int rows = min(GROUP_ROWS, p.row_tiles - g * GROUP_ROWS);
  ct = r / rows;
  rt = g * GROUP_ROWS + (r - ct * rows);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Column c of a group's W, counted from the group's first one.
template <bool SEG>
__host__ __device__ __forceinline__ constexpr int column(int c) {
  return SEG && c >= 64 ? c + 64 : c;
}

template <int OUT>
__device__ __forceinline__ void store_one(void* row, int col, float v) {
  if (OUT == OUT_BF16) static_cast<__nv_bfloat16*>(row)[col] = __float2bfloat16_rn(v);
  if (OUT == OUT_F16) static_cast<__half*>(row)[col] = __float2half_rn(v);
  if (OUT == OUT_F32) static_cast<float*>(row)[col] = v;
}

// Output goes through shared memory in boxes of 32 rows, 128 or 64 bytes wide, in the tensor map's swizzled order:
// 16-byte piece q of row r at piece q ^ (r mod 8) of 128, q ^ (r / 2 mod 4) of 64 bytes. No bank conflicts either way.
__host__ __device__ constexpr int out_row_bytes(int bytes) { return bytes >= 128 ? 128 : 64; }
template <int ROW>
__device__ __forceinline__ int swizzled(int r, int q) {
  return r * ROW + ((ROW == 128 ? q ^ (r & 7) : q ^ ((r >> 1) & 3)) << 4);
}

// Writes a warp's 32 rows x W columns of y at (m0, n0), up to 128 bytes a row at a time through one of two 4 KB
// buffers: a tensor-map store that runs on while the warp goes back to its next tile (rows beyond M and columns
// beyond N are clipped by the copy), or, where y's base or rows are not 16-byte aligned, plain coalesced stores.
// Straight from registers, 32 rows an instruction, the same tile took 6400 clocks of the 10240 that its MMAs
// take at K = 2560; in boxes of 64 bytes the product above takes 215 us instead of 208.
template <int OUT, int W, bool SEG>
__device__ __forceinline__ void store_rows(const Product& p, const CUtensorMap* ymap, char* bufs, int& turn, int m0,
                                           int n0, int lane, const float2 (&acc)[W / 2]) {
  constexpr int ES = OUT == OUT_F32 ? 4 : 2;
  constexpr int ROW = out_row_bytes(W * ES), CC = ROW / ES, Q = ROW / 16;   // bytes, columns and 16-byte pieces of a row
#pragma unroll
  for (int c = 0; c < W; c += CC, ++turn) {
    char* buf = bufs + (turn & (OUT_BUFS - 1)) * OUT_BUF;
    const int n = n0 + column<SEG>(c);
    if (lane == 0) bulk_wait_read<OUT_BUFS - 1>();   // this buffer's last store has been read
    __syncwarp();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      uint32_t v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (OUT == OUT_F32) v[i] = __float_as_uint(i & 1 ? acc[(c + 4 * q + i) / 2].y : acc[(c + 4 * q + i) / 2].x);
        if (OUT == OUT_BF16) v[i] = pack_bf16(acc[c / 2 + 4 * q + i].x, acc[c / 2 + 4 * q + i].y);
        if (OUT == OUT_F16) v[i] = pack_f16(acc[c / 2 + 4 * q + i].x, acc[c / 2 + 4 * q + i].y);
      }
      *reinterpret_cast<uint4*>(buf + swizzled<ROW>(lane, q)) = make_uint4(v[0], v[1], v[2], v[3]);
    }
    if (p.tma_out) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (n < p.N) tma_store_2d(ymap, n, m0, smem_u32(buf));
        bulk_commit();
      }
    } else {
      __syncwarp();
      char* y = static_cast<char*>(p.y);
#pragma unroll 4
      for (int i = lane; i < 32 * CC; i += 32) {
        const int r = i / CC, col = i % CC;
        if (m0 + r < p.M && n + col < p.N) {
          const char* from = buf + swizzled<ROW>(r, col * ES >> 4) + (col * ES & 15);
          char* to = y + ((long long)(m0 + r) * p.ldy + n + col) * ES;
          if (ES == 4)
            *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
          else
            *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
        }
      }
      __syncwarp();
    }
  }
}

// A row's statistics over the W values of a group whose first column is n, and its token's logit if it is one.
// Columns beyond N become -inf, which adds nothing.
template <int W, bool SEG>
__device__ __forceinline__ LogitStat row_stats(const Product& p, int m, int n, float2 (&acc)[W / 2]) {
  if (n + column<SEG>(W - 1) >= p.N) {
#pragma unroll
    for (int c = 0; c < W; c += 2) {
      if (n + column<SEG>(c) >= p.N) acc[c / 2].x = -INFINITY;
      if (n + column<SEG>(c + 1) >= p.N) acc[c / 2].y = -INFINITY;
    }
  }
  const long long id = p.ids[m] - n;
  if (id >= 0 && id <= column<SEG>(W - 1) && id < p.N - n) {
    uint32_t bits = 0;                               // (an indexed read would move the values to memory)
    bool mine = false;
#pragma unroll
    for (int c = 0; c < W; ++c) {
      const bool hit = column<SEG>(c) == (int)id;
      bits |= __float_as_uint(c & 1 ? acc[c / 2].y : acc[c / 2].x) & (hit ? 0xffffffffu : 0u);
      mine |= hit;
    }
    if (mine) p.token[m] = __uint_as_float(bits);
  }
  // y = (x - m) log2 e as one fused multiply-add, x log2 e - R with R = m log2 e rounded; the sums are moved from R
  // to m at the end. (A multiplication and a subtraction each, scalar, took 1640 us for 1540 at 4096 x 151936 x 2560.)
  LogitStat st;
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < W / 2; ++c) mx[c & 3] = max3(mx[c & 3], acc[c].x, acc[c].y);
  st.m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
  const float ref = st.m == -INFINITY ? 0.f : st.m;
  float moved = ref * LOG2E, rest = fmaf(ref, LOG2E, -moved);
  if (!(fabsf(ref) < LARGE)) {                       // there R is too coarse
    const float2 by = make_float2(-ref, -ref);
#pragma unroll
    for (int c = 0; c < W / 2; ++c) acc[c] = add2(acc[c], by);
    moved = rest = 0.f;
  }
  const float2 l2 = make_float2(LOG2E, LOG2E), r2 = make_float2(-moved, -moved);
  float2 s[2] = {}, w[2] = {};
#pragma unroll
  for (int c = 0; c < W / 2; ++c) {
    float2 y = fma2(acc[c], l2, r2);
    y = make_float2(max_nan(y.x, LOWEST_Y), max_nan(y.y, LOWEST_Y));
    const float2 x = make_float2(exp2_approx(y.x), exp2_approx(y.y));
    s[c & 1] = add2(s[c & 1], x);
    w[c & 1] = fma2(x, y, w[c & 1]);
  }
  const float total = (s[0].x + s[0].y) + (s[1].x + s[1].y), weighted = (w[0].x + w[0].y) + (w[1].x + w[1].y);
  const float back = exp2_approx(-rest);
  st.s = total * back;
  st.w = fmaf(-rest, total, weighted) * back * LN2;
  if (isnan(st.s)) st = LogitStat{0.f, NAN, NAN};    // a NaN, or +inf (whose difference from itself is NaN)
  return st;
}

// Shared memory: barriers | factors | output buffers or statistics | ring of stages, each the token rows and the
// weight rows. Where one row tile holds all tokens (few), only the quarters of 32 rows that hold some have output
// buffers and a stage holds only those rows, which leaves more stages for the weight (8 rows: 6 for 4, 67 us for 73
// at 8 x 151936 x 2560); the MMAs then read on past them, into rows of the accumulator that nobody looks at.
__host__ __device__ constexpr int out_offset() { return (1024 + 2 * FGROUP * F_LD * 4 + 1023) / 1024 * 1024; }
template <int OUT>
__host__ __device__ constexpr int ring_offset(int quarters) {
  return out_offset() + (OUT == OUT_STATS ? 2 * 3 * EPI_GROUPS * BM * 4 : EPI_GROUPS * quarters * OUT_BUFS * OUT_BUF);
}

// One CTA (CG = 1; gridDim / cluster size clusters, whose CTAs split K) or one CTA pair (CG = 2).
template <int CG, int BN, int OUT>
__global__ void __launch_bounds__(THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                   const __grid_constant__ CUtensorMap ymap, Product p) {
  constexpr int W = Tile<BN>::W, NBUF = Tile<BN>::NBUF, UNITS = Tile<BN>::UNITS, UN = Tile<BN>::UN;
  constexpr bool SEG = CG == 2 && UNITS == 2;                      // a group's columns: 64 of each 128-column block
  constexpr int B_ROWS = BN / CG;                    // weight rows in this CTA's shared memory
  const int quarters = CG == 1 ? p.quarters : 4, A_BYTES = CG == 1 ? p.a_bytes : BM * 128;
  const int STAGE = A_BYTES + B_ROWS * 128;
  constexpr bool CAN_SPLIT = CG == 1 && OUT != OUT_STATS && !Tile<BN>::SPLIT_REGS;
  extern __shared__ char sm_raw[];
  char* sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* acc_full = empty + MAX_STAGES;
  uint64_t* acc_empty = acc_full + 8;
  uint64_t* f_full = acc_empty + 8;
  uint64_t* f_empty = f_full + 2;
  uint64_t* done = f_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 2);
  float* factors = reinterpret_cast<float*>(sm + 1024);
  float* stat_s = reinterpret_cast<float*>(sm + out_offset());      // head: [2][3][EPI_GROUPS][BM]
  char* ring = sm + ring_offset<OUT>(quarters);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = cluster_rank(), csize = cluster_size();
  const uint32_t split = CAN_SPLIT ? csize : 1, part = CAN_SPLIT ? crank : 0;
  const int KB = (p.K + 127) >> 7;
  const int kb0 = KB * part / split, kb1 = KB * (part + 1) / split;
  const int tiles = p.row_tiles * p.col_tiles;
  const int first = blockIdx.x / csize, step = gridDim.x / csize;
  const int nstage = p.nstage;

  // The copies' place in the CTA's blocks: thread 0 alone moves it.
  const uint32_t rank = CG == 2 ? crank : 0;
  struct {
    int t, kb, m, n, s, round;
    long long count;
  } at;
  auto to_tile = [&](int t) {
    int rt, ct;
    tile_at(p, t, rt, ct);
    at.t = t;
    at.kb = kb0;
    at.m = (rt * CG + (int)rank) * BM;
    at.n = ct * BN + (int)rank * B_ROWS;
  };
  auto copy_next = [&]() {                           // the next block into stage at.s, which is free
    uint32_t bar = smem_u32(&full[at.s]);
    if (CG == 1 || rank == 0) mbar_arrive_expect_tx(&full[at.s], (uint32_t)(p.box_m + B_ROWS) * 128 * CG);
    if (CG == 2) bar = map_to_rank(bar, 0);
    const uint32_t dst = smem_u32(ring + at.s * STAGE);
    tma_load_2d<CG>(dst, &xmap, at.kb * 128, at.m, bar);
    if (p.packed)
      tma_load_4d<CG>(dst + A_BYTES, &wmap, 0, 0, at.n / 16, at.kb, bar);
    else
      tma_load_2d<CG>(dst + A_BYTES, &wmap, at.kb * 128, at.n, bar);
    ++at.count;
    if (++at.s == nstage) at.s = 0, ++at.round;
    if (++at.kb == kb1) {
      at.t += step;
      if (at.t < tiles) to_tile(at.t);
    }
  };
  if (CG == 1 && csize > 1) cluster_arrive();        // (waited for before the first store to another CTA)
  if (threadIdx.x == 0) {
    prefetch_map(&xmap);
    prefetch_map(&wmap);
    for (int i = 0; i < nstage; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], UNITS);                   // a commit of each issuer that reads the stage
    }
    for (int i = 0; i < NBUF; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], Tile<BN>::RELEASERS * CG);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&f_full[i], 1);
      mbar_init(&f_empty[i], EPI_WARPS);
    }
    mbar_init(&done[0], 1);
    mbar_init(&done[1], 1);
    fence_mbar_init();
    at.s = at.round = 0;
    at.count = 0;
    to_tile(first);
    // The first ring of copies goes out before the rest of the CTA is set up (a pair's needs the other CTA's barriers).
    if (CG == 1)
      while (at.t < tiles && at.round == 0) copy_next();
  }
  if (warp == 1) tmem_alloc_512<CG>(tmem_slot);
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (OUT == OUT_STATS) griddep_launch_dependents();  // the merge may take its place as SMs free up

  float2 acc[W / 2];
  if (Tile<BN>::SPLIT_REGS && warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Tile<BN>::OTHER_REGS));
  if (warp == 0) {
    if (lane == 0) {
      // ---------------- copies ----------------
      bool ok = true;
      while (at.t < tiles && ok) {
        ok = at.round == 0 || mbar_wait_limited(&empty[at.s], (at.round - 1) & 1, p.tries);
        if (ok) copy_next();
      }
      // Leave only when this CTA's copies have landed and been read: the MMAs' commit of each stage's last use.
      const long long oldest = at.count > nstage ? at.count - nstage : 0;
      for (long long q = oldest; q < at.count && ok; ++q)
        ok = mbar_wait_limited(&empty[q % nstage], (uint32_t)(q / nstage) & 1, p.tries);
      if (!ok) {
        atomicExch(&g_score_err, 1);
        if (CG == 1 || rank == 0)
          for (long long q = oldest; q < at.count; ++q)
            mbar_wait_limited(&full[q % nstage], (uint32_t)(q / nstage) & 1, WAIT_TRIES);
        else                                           // the pair's barriers are the other CTA's: time for any copy to land
          for (const uint64_t t0 = globaltimer_ns(); globaltimer_ns() - t0 < 10000000ull;) __nanosleep(1000);
      }
    }
    __syncwarp();
  } else if (warp == 1 || warp == 3) {
    if (CG == 1 || crank == 0) {
      // ---------------- MMAs ----------------
      // Two issuers, since a block's wait, four MMAs and two commits take a warp about 500 clocks: of a block's two
      // accumulators one each (BN = 256), else every other block. The whole warp walks the loop and one elected
      // lane issues.
      const uint32_t idesc = (1u << 4)                             // D: f32
                             | ((uint32_t)(UN >> 3) << 17)         // N
                             | ((uint32_t)(BM * CG >> 4) << 24);   // M; A, B: e4m3, K-major
      const int u = warp >> 1;
      constexpr int STEP = UNITS == 2 ? 1 : 2;                     // blocks
      const uint32_t b_offset = UNITS == 2 ? u * (UN / CG * 128) : 0;
      const long long blocks = first < tiles ? (long long)((tiles - first + step - 1) / step) * (kb1 - kb0) : 0;
      int s = UNITS == 2 ? 0 : u, round = 0, buf = u, use = 0;
      if (s >= nstage) s -= nstage, ++round;
      bool ok = true;
      for (long long i = UNITS == 2 ? 0 : u; i < blocks; i += STEP) {
        ok = warp_wait(&full[s], round & 1, &acc_empty[buf], (use - 1) & 1, use > 0, p.tries);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t st = smem_u32(ring + s * STAGE);
          const uint64_t a = sw128_desc(st), b = sw128_desc(st + A_BYTES + b_offset);
          const uint32_t d = tmem + buf * UN;
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_f8<CG>(d, a + 2 * k, b + 2 * k, idesc, k > 0 ? 1u : 0u);
          tc_commit<CG>(&acc_full[buf]);
          tc_commit<CG>(&empty[s]);
        }
        __syncwarp();
        s += STEP;
        if (s >= nstage) s -= nstage, ++round;
        buf += 2;
        if (buf >= NBUF) buf -= NBUF, ++use;
      }
      if (!ok) {                                       // what was issued still writes TMEM
        if (elect_one()) {
          atomicExch(&g_score_err, 1);
          tc_commit<CG>(&done[u]);
        }
        __syncwarp();
        mbar_wait_limited(&done[u], 0, WAIT_TRIES);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---------------- factors ----------------
    // Lane = (row mod 8, block of the group): row-major scales are read 16 B a row, four blocks in one pass.
    const int r8 = lane >> 2, i = lane & 3;
    int fg = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      int rt, ct;
      tile_at(p, t, rt, ct);
      const int m = (rt * CG + (int)rank) * BM + r8, nb = ct * BN >> 7;
      for (int kb = kb0; kb < kb1; kb += FGROUP, ++fg) {
        float x[BM / 8], w[Tile<BN>::BLOCKS];
#pragma unroll
        for (int b = 0; b < Tile<BN>::BLOCKS; ++b)
          w[b] = kb + i < kb1 && (nb + b) * 128 < p.N ? __ldg(p.ws + (long long)(nb + b) * p.ws_row + kb + i) : 0.f;
#pragma unroll
        for (int j = 0; j < BM / 8; ++j)
          x[j] = kb + i < kb1 && m + 8 * j < p.M
                     ? __ldg(p.xs + (long long)(m + 8 * j) * p.xs_row + (long long)(kb + i) * p.xs_col) : 0.f;
        if (fg >= 2) ok = warp_wait(&f_empty[fg & 1], ((fg >> 1) - 1) & 1, p.tries);
        if (!ok) break;
        float* dst = factors + ((fg & 1) * FGROUP + i) * F_LD + r8;
#pragma unroll
        for (int b = 0; b < Tile<BN>::BLOCKS; ++b)
#pragma unroll
          for (int j = 0; j < BM / 8; ++j) dst[b * BM + 8 * j] = x[j] * w[b];
        __syncwarp();
        if (lane == 0) mbar_arrive(&f_full[fg & 1]);
      }
    }
    if (!ok && lane == 0) atomicExch(&g_score_err, 1);
  } else if (warp >= 4) {
    // ---------------- promotion and output ----------------
    if constexpr (Tile<BN>::SPLIT_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Tile<BN>::EPI_REGS));
    const int quarter = warp & 3, group = (warp >> 2) - 1;
    const uint32_t lanes = tmem + ((uint32_t)(32 * quarter) << 16) + (UNITS == 1 ? group * W : 0);
    const int row_in_tile = 32 * quarter + lane;
    const float* my_factors = factors + (BN == 256 && !SEG ? group : 0) * BM + row_in_tile;
    const int col = SEG ? 64 * group : W * group;    // first column of the group in its tile
    const uint32_t release = map_to_rank(smem_u32(acc_empty), CG == 2 ? 0 : cluster_rank());   // where the MMAs are issued
    int buf = UNITS == 2 ? group : 0, use = 0, turn = 0, fg = 0;
    bool ok = true;
    for (int t = first; t < tiles; t += step) {
      int rt, ct;
      tile_at(p, t, rt, ct);
      const int m = (rt * CG + (int)rank) * BM + row_in_tile, n = ct * BN + col;
#pragma unroll
      for (int c = 0; c < W / 2; ++c) acc[c] = make_float2(0.f, 0.f);
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        const int fi = (kb - kb0) & (FGROUP - 1);
        ok = warp_wait(&acc_full[buf], use & 1, &f_full[fg & 1], (fg >> 1) & 1, fi == 0, p.tries);
        if (!ok) break;
        tc_fence_after();
        const float* now = my_factors + ((fg & 1) * FGROUP + fi) * F_LD;
        const float scale0 = now[0], scale1 = SEG ? now[BM] : scale0;
        const uint32_t src = lanes + buf * UN;
        constexpr int C = 16;                        // columns of one TMEM load (32: 204 us for 201 above)
#pragma unroll
        for (int c = 0; c < W; c += C) {
          uint32_t v[C];
          tmem_ld16(src + c, v);
          tmem_wait_ld16(v);
          if (c + C == W) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(release + buf * 8);
          }
#pragma unroll
          for (int i = 0; i < C / 2; ++i) fma2_scaled(acc[c / 2 + i], v[2 * i], v[2 * i + 1], c < 64 ? scale0 : scale1);
        }
        if (fi == FGROUP - 1 || kb + 1 == kb1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&f_empty[fg & 1]);
          ++fg;
        }
        buf += UNITS;
        if (buf >= NBUF) buf -= NBUF, ++use;
      }
      if (!ok) {                                       // a wait ran out: this tile and the rest come out NaN
#pragma unroll
        for (int c = 0; c < W / 2; ++c) acc[c] = make_float2(NAN, NAN);
      }
      if constexpr (OUT == OUT_STATS) {
        // a tile's four column groups leave one set of statistics
        float* own = stat_s + (turn & 1) * 3 * EPI_GROUPS * BM + row_in_tile;
        LogitStat st = logit_stat_empty();
        if (m < p.M && n < p.N) st = row_stats<W, SEG>(p, m, n, acc);
        own[(0 * EPI_GROUPS + group) * BM] = st.m;
        own[(1 * EPI_GROUPS + group) * BM] = st.s;
        own[(2 * EPI_GROUPS + group) * BM] = st.w;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * EPI_WARPS) : "memory");
        if (group == 0 && m < p.M) {
#pragma unroll
          for (int g = 1; g < EPI_GROUPS; ++g)
            st = logit_stat_merge(st, LogitStat{own[g * BM], own[(EPI_GROUPS + g) * BM], own[(2 * EPI_GROUPS + g) * BM]});
          p.part[(long long)m * p.col_tiles + ct] = make_float4(st.m, st.s, st.w, 0.f);
        }
        ++turn;
      } else if (split == 1 && n < p.N && m - lane < p.M) {
        store_rows<OUT, W, SEG>(p, &ymap, sm + out_offset() + (group * quarters + quarter) * OUT_BUFS * OUT_BUF, turn,
                                m - lane, n, lane, acc);
      }
    }
    if (OUT != OUT_STATS && lane == 0) bulk_wait_all();
    if (!ok && lane == 0) atomicExch(&g_score_err, 1);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CAN_SPLIT) {
    // ---------------- K split over the cluster's CTAs: one tile ----------------
    // Each CTA owns BN / split of the columns: the others push their sums of those into its output buffers, which
    // nothing else uses here, and it adds them in rank order.
    if (split > 1) {
      const int share = BN / split;
      float* sums = reinterpret_cast<float*>(sm + out_offset());       // [split][32 quarters][share]
      static_assert(32 * BN * 4 <= EPI_GROUPS * OUT_BUFS * OUT_BUF, "the output buffers hold a tile");
      const int cap = 32 * quarters;
      int rt, ct;
      tile_at(p, first, rt, ct);
      const int rows = min(BM, p.M - rt * BM);
      cluster_wait();                                // every CTA has started
      if (warp >= 4) {
        const int group = (warp >> 2) - 1, r = 32 * (warp & 3) + lane;
        if (r < rows) {
#pragma unroll
          for (int c = 0; c < W; c += 4) {
            const int col = group * W + c, owner = col / share;
            st_cluster_f4(map_to_rank(smem_u32(sums + (part * cap + r) * share + col - owner * share), owner),
                          make_float4(acc[c / 2].x, acc[c / 2].y, acc[c / 2 + 1].x, acc[c / 2 + 1].y));
          }
        }
      }
      cluster_sync_all();
      const int quads = share / 4;
      for (int e = threadIdx.x; e < rows * quads; e += THREADS) {
        const int r = e / quads, c = (e - r * quads) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t q = 0; q < split; ++q) {
          const float4 u = *reinterpret_cast<const float4*>(sums + (q * cap + r) * share + c);
          v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        }
        const int n = ct * BN + part * share + c;
        char* to = static_cast<char*>(p.y) + ((long long)(rt * BM + r) * p.ldy + n) * (OUT == OUT_F32 ? 4 : 2);
        if (n + 4 <= p.N && p.tma_out) {
          if (OUT == OUT_F32) *reinterpret_cast<float4*>(to) = v;
          if (OUT == OUT_BF16) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
          if (OUT == OUT_F16) *reinterpret_cast<uint2*>(to) = make_uint2(pack_f16(v.x, v.y), pack_f16(v.z, v.w));
        } else {
          if (n < p.N) store_one<OUT>(to, 0, v.x);
          if (n + 1 < p.N) store_one<OUT>(to, 1, v.y);
          if (n + 2 < p.N) store_one<OUT>(to, 2, v.z);
          if (n + 3 < p.N) store_one<OUT>(to, 3, v.w);
        }
      }
    }
  }
  if (CG == 2) cluster_sync_all();                 // the other CTA may still signal this one's barriers
  tc_fence_after();
  if (warp == 1) tmem_dealloc_512<CG>(tmem);
}

// One CTA per row: the column tiles' statistics merged. Launched as the product's programmatic dependent.
constexpr int MERGE_THREADS = 128;
__global__ void __launch_bounds__(MERGE_THREADS)
    head_merge_kernel(const float4* __restrict__ part, const float* __restrict__ token,
                      const long long* __restrict__ ids, int tiles, int N, float* logprob, float* entropy, float* lse) {
  __shared__ LogitStat sh[MERGE_THREADS / 32];
  const int m = blockIdx.x;
  const long long id = ids[m];
  griddep_wait();
  LogitStat st = logit_stat_empty();
  for (int t = threadIdx.x; t < tiles; t += MERGE_THREADS) {
    const float4 o = part[(long long)m * tiles + t];
    st = logit_stat_merge(st, LogitStat{o.x, o.y, o.z});
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
    st = logit_stat_merge(st, LogitStat{__shfl_xor_sync(~0u, st.m, o), __shfl_xor_sync(~0u, st.s, o),
                                        __shfl_xor_sync(~0u, st.w, o)});
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = st;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < MERGE_THREADS / 32; ++i) st = logit_stat_merge(st, sh[i]);
    const bool valid = id >= 0 && id < N;
    const RowResult r = logit_stat_finish(st, valid ? token[m] : 0.f, valid);
    logprob[m] = r.logprob;
    entropy[m] = r.entropy;
    lse[m] = r.lse;
  }
}

// ---- host -----------------------------------------------------------------------------------------

struct Operands {
  const void* x;
  long long ldx;
  const float* xs;
  long long xs_row, xs_col;
  const void* w;
  long long ldw;
  int packed;
  const float* ws;
  long long ws_row;
  int M, N, K;
};

bool aligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_operands(const Operands& p) {
  if (p.M < 0 || p.M > (1 << 30)) return -1;         // (coordinates and tile numbers are 32-bit)
  if (p.N < 1 || p.N > (1 << 30) || (p.packed && p.N % 16)) return -2;
  if (p.K < 16 || p.K > (1 << 30) || p.K % 16 || (p.packed && p.K % 128)) return -3;
  if (p.ldx < p.K || p.ldx % 16 || (!p.packed && (p.ldw < p.K || p.ldw % 16))) return -4;
  if (!aligned(p.x, 16) || !aligned(p.w, 16)) return -10;
  return 0;
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

// rows x K bytes, row-major: boxes of box_rows x 128 B landing as [box_rows][128 B], 128-byte swizzled.
int rows_map(CUtensorMap* m, const void* base, int rows, int K, long long ld, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, es[2] = {1, 1};
  const auto fn = encoder();
  if (fn == nullptr) return -12;
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -12;
}

// The strip pack [N/16][K/128][16 rows][128 B], already swizzled: (byte, row, strip, 128-K block).
int strips_map(CUtensorMap* m, const void* base, int N, int K, int box_rows) {
  const int KB = K / 128;
  const cuuint64_t dims[4] = {128, 16, (cuuint64_t)(N / 16), (cuuint64_t)KB};
  const cuuint64_t strides[3] = {128, (cuuint64_t)KB * 2048, 2048};
  const cuuint32_t box[4] = {128, 16, (cuuint32_t)(box_rows / 16), 1}, es[4] = {1, 1, 1, 1};
  const auto fn = encoder();
  if (fn == nullptr) return -12;
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -12;
}

// y [rows, cols] of 2 or 4-byte elements: boxes of 32 rows x row_bytes, swizzled.
int out_map(CUtensorMap* m, void* base, int rows, int cols, long long ld, int es, int row_bytes) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? ld * es : ((long long)cols * es + 15) / 16 * 16)};
  const cuuint32_t box[2] = {(cuuint32_t)(row_bytes / es), 32}, one[2] = {1, 1};
  const auto fn = encoder();
  if (fn == nullptr) return -12;
  return fn(m, es == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base, dims, strides, box,
            one, CU_TENSOR_MAP_INTERLEAVE_NONE, row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -12;
}

// Tries of a pipeline wait: WAIT_TRIES, or what the environment says when the first call is made.
uint32_t wait_tries() {
  static const uint32_t n = [] {
    const char* s = std::getenv("B200_SCORE_WAIT_TRIES");
    return s != nullptr && *s >= '0' && *s <= '9' ? (uint32_t)std::strtoul(s, nullptr, 10) : WAIT_TRIES;
  }();
  return n;
}

constexpr int MAX_DEVICES = 64;

int num_sms(int dev) {
  static int cached[MAX_DEVICES] = {};
  int n = 0;
  if (dev < 0 || dev >= MAX_DEVICES) return 148;
  if (cached[dev] <= 0)
    cached[dev] = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
  return cached[dev];
}

// Raises the kernel's shared-memory limit, once per device, and checks what its register split relies on.
template <int CG, int BN, int OUT>
int make_ready(int dev) {
  static bool ready[MAX_DEVICES] = {};
  if (dev < MAX_DEVICES && ready[dev]) return 0;
  const void* kern = reinterpret_cast<const void*>(product_kernel<CG, BN, OUT>);
  if (Tile<BN>::SPLIT_REGS) {                         // the split's sum must be what the launch brings
    cudaFuncAttributes fa;
    const cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return (int)e;
    if (fa.numRegs != Tile<BN>::LAUNCH_REGS) return -13;
  }
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_CAP);
  if (e == cudaSuccess && dev < MAX_DEVICES) ready[dev] = true;
  return (int)e;
}

// How many clusters of `split` CTAs the device holds at once (fewer than its SMs / split: a cluster stays within a
// group of SMs), asked once per device.
template <int BN, int OUT>
int clusters_at_once(int dev, int split) {
  static int cached[MAX_DEVICES][4] = {};
  if (split == 1) return num_sms(dev);
  const int at = split == 2 ? 1 : split == 4 ? 2 : 3;
  if (dev < MAX_DEVICES && cached[dev][at] > 0) return cached[dev][at];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(num_sms(dev) / split * split);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM_MIN;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (make_ready<1, BN, OUT>(dev) != 0 ||
      cudaOccupancyMaxActiveClusters(&n, product_kernel<1, BN, OUT>, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();                               // the launch itself will say what is wrong
    return num_sms(dev) / split * 3 / 4;
  }
  if (dev < MAX_DEVICES) cached[dev][at] = n;
  return n;
}

template <int CG, int BN, int OUT>
int launch(const Operands& o, Product p, int dev, int split, cudaStream_t stream) {
  constexpr int B_ROWS = BN / CG;
  p.xs = o.xs, p.xs_row = o.xs_row, p.xs_col = o.xs_col, p.ws = o.ws, p.ws_row = o.ws_row;
  p.M = o.M, p.N = o.N, p.K = o.K, p.packed = o.packed;
  p.tries = wait_tries();
  p.box_m = std::min(BM, (o.M + 7) / 8 * 8);
  p.row_tiles = (o.M + BM * CG - 1) / (BM * CG);
  p.col_tiles = (o.N + BN - 1) / BN;
  if ((long long)p.row_tiles * p.col_tiles > (1 << 30)) return -8;
  CUtensorMap xmap, wmap, ymap{};
  int rc = rows_map(&xmap, o.x, o.M, o.K, o.ldx, p.box_m);
  if (rc == 0) rc = o.packed ? strips_map(&wmap, o.w, o.N, o.K, B_ROWS) : rows_map(&wmap, o.w, o.N, o.K, o.ldw, B_ROWS);
  if (rc == 0 && OUT != OUT_STATS && p.tma_out) rc = out_map(&ymap, p.y, o.M, o.N, p.ldy, OUT == OUT_F32 ? 4 : 2,
                                                             out_row_bytes(Tile<BN>::W * (OUT == OUT_F32 ? 4 : 2)));
  if (rc != 0) return rc;
  const int tiles = p.row_tiles * p.col_tiles, KB = (o.K + 127) / 128;
  const int cl = CG == 2 ? 2 : split;
  // As few CTAs (pairs) as take no more turns than all SMs would: 8 x 151936 x 2560, whose 594 tiles are four turns and
  // two tiles of 148 SMs, takes 73 us on 119 and 76 on 148.
  const int turns = split > 1 ? 1 : (tiles + num_sms(dev) / cl - 1) / (num_sms(dev) / cl);
  const int clusters = (tiles + turns - 1) / turns;
  const int per_cta = split > 1 ? (KB + split - 1) / split : turns * KB;
  const bool few = CG == 1 && p.row_tiles == 1;
  p.quarters = few ? (o.M + 31) / 32 : 4;
  p.a_bytes = few ? p.box_m * 128 : BM * 128;
  const int stage = p.a_bytes + B_ROWS * 128;
  // alignment, all before the ring, what the MMAs read past its end
  const int fixed = 1024 + ring_offset<OUT>(p.quarters) + (BM * 128 - p.a_bytes);
  p.nstage = std::min({MAX_STAGES, (SMEM_CAP - fixed) / stage, std::max(2, per_cta)});
  const int smem = std::max(SMEM_MIN, fixed + p.nstage * stage);
  auto kern = product_kernel<CG, BN, OUT>;
  rc = make_ready<CG, BN, OUT>(dev);
  if (rc != 0) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * cl);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, xmap, wmap, ymap, p);
  return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

constexpr int HEAD_BN = 256;                        // columns of a head tile, which leave one set of statistics a row
int head_tiles(int N) { return (N + HEAD_BN - 1) / HEAD_BN; }

template <int OUT>
int launch_product(const Operands& o, const Product& p, cudaStream_t stream) {
  // Columns of a tile (256: of a CTA pair's, above 128 rows) and CTAs that split its K, by the time they take: a
  // start, the busiest SM's 128-K blocks, and with K split the sums' way to their owners, in measured microseconds.
  // Measured there, chosen first: 5 x 2560 x 2560 at (128, 4) 7.2, (64, 2) 8.0, (64, 1) 9.7; 512 x 1024 x 2560 at
  // (64, 1) 9.7, (64, 2) 9.9, (128, 4) 12.2; 16 x 10240 x 2560 at (128, 1) 11.9, (64, 1) 16.6; 8192 x 10240 x 2560
  // at 256 columns 201, (128, 1) 300. K is split only as far as all clusters run at once: counted by SMs alone,
  // 1 x 1024 x 2560 and 64 x 1024 x 2560 took 8 CTAs a tile and a second turn, 9.8 and 12.0 for 6.1 and 7.4.
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  const int KB = (o.K + 127) / 128, sms = num_sms(dev);
  int bn = 256, split = 1;
  double best = 1e300;
  auto consider = [&](int b, int s, long long ctas, int at_once, double start, double block) {
    if (s > KB || (s > 1 && ctas > at_once)) return;
    const double sums = s > 1 ? 1.2 + std::min(o.M, BM) * (b / 64) * 0.015 : 0.;
    const double us = start + (double)((ctas + at_once - 1) / at_once) * ((KB + s - 1) / s) * block + sums;
    if (us < best) best = us, bn = b, split = s;
  };
  const long long rows = (o.M + BM - 1) / BM;
  if (rows > 1)
    consider(256, 1, (rows + 1) / 2 * ((o.N + 255) / 256), sms / 2, 5.0, 0.56);
  else
    consider(256, 1, (o.N + 255) / 256, sms, 5.0, 0.50);
  if constexpr (OUT != OUT_STATS)
    for (int s = 1; s <= 8; s *= 2) {
      consider(128, s, rows * ((o.N + 127) / 128) * s, clusters_at_once<128, OUT>(dev, s) * s, 4.6, 0.40);
      consider(64, s, rows * ((o.N + 63) / 64) * s, clusters_at_once<64, OUT>(dev, s) * s, 3.6, 0.31);
    }
  if (bn == 256) return o.M > BM ? launch<2, 256, OUT>(o, p, dev, 1, stream) : launch<1, 256, OUT>(o, p, dev, 1, stream);
  if constexpr (OUT != OUT_STATS)
    return bn == 128 ? launch<1, 128, OUT>(o, p, dev, split, stream) : launch<1, 64, OUT>(o, p, dev, split, stream);
  return -8;
}

}  // namespace

extern "C" {

int b200_fp8_block_gemm(const void* qx, long long ldx, const float* xs, long long xs_row, long long xs_col,
                        const void* wq, long long ldw, int packed, const float* ws, long long ws_row, void* y,
                        long long ldy, int y_dtype, int M, int N, int K, cudaStream_t stream) {
  const Operands o{qx, ldx, xs, xs_row, xs_col, wq, ldw, packed, ws, ws_row, M, N, K};
  const int rc = check_operands(o);
  if (rc != 0) return rc;
  if (ldy < N) return -4;
  if (y_dtype < 0 || y_dtype > 2) return -5;
  const int es = y_dtype == 2 ? 4 : 2;
  if (!aligned(y, es)) return -10;
  if (M == 0) return 0;
  Product p{};
  p.y = y;
  p.ldy = ldy;
  p.tma_out = aligned(y, 16) && (M == 1 || ldy * es % 16 == 0);
  return y_dtype == 0 ? launch_product<OUT_BF16>(o, p, stream)
                      : y_dtype == 1 ? launch_product<OUT_F16>(o, p, stream) : launch_product<OUT_F32>(o, p, stream);
}

long long b200_fp8_head_logprobs_workspace_bytes(int M, int N) {
  if (M <= 0 || N <= 0) return 0;
  return (16LL * head_tiles(N) + 4) * M;
}

int b200_fp8_head_logprobs(const void* qx, long long ldx, const float* xs, long long xs_row, long long xs_col,
                           const void* wq, long long ldw, int packed, const float* ws, long long ws_row,
                           const long long* ids, int M, int N, int K, float* logprob, float* entropy, float* lse,
                           void* workspace, long long workspace_bytes, cudaStream_t stream) {
  const Operands o{qx, ldx, xs, xs_row, xs_col, wq, ldw, packed, ws, ws_row, M, N, K};
  int rc = check_operands(o);
  if (rc != 0) return rc;
  if (M == 0) return 0;
  if (workspace == nullptr || workspace_bytes < b200_fp8_head_logprobs_workspace_bytes(M, N)) return -9;
  if (!aligned(workspace, 16)) return -10;
  Product p{};
  p.ids = ids;
  p.part = static_cast<float4*>(workspace);
  p.token = reinterpret_cast<float*>(p.part + (long long)M * head_tiles(N));
  rc = launch_product<OUT_STATS>(o, p, stream);
  if (rc != 0) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(M);
  cfg.blockDim = dim3(MERGE_THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, head_merge_kernel, (const float4*)p.part, (const float*)p.token, ids,
                                           head_tiles(N), N, logprob, entropy, lse);
  return (int)(e != cudaSuccess ? e : cudaGetLastError());
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
