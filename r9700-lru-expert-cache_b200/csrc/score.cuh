// Shared pieces of the scoring kernels (fp8_gemm.cu, logprobs.cu).
#pragma once
#include "common.cuh"

namespace b200 {

// Programmatic dependent launch: the dependent grid may be placed while its primary still runs; griddep_wait()
// returns once the primary is complete and its writes are visible.
B200_DEVINL void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
B200_DEVINL void griddep_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The larger one; NaN if either is.
B200_DEVINL float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

B200_DEVINL float max3(float a, float b, float c) {   // ignores NaN
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// Beyond this size a logit times log2 e is known to no better than a few units, or out of fp32's range: below
// -LARGE a logit is not taken as a reference (beside any other it has no weight), and a row whose largest logit is
// not within +-LARGE is done again in natural units.
constexpr float LARGE = 4e7f;
constexpr float LOWEST_Y = -160.f;         // 2^-160 = 0 in fp32, and 0 * -160 = 0 where 0 * -inf is not

B200_DEVINL float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// (a.x + b.x, a.y + b.y) and a fused multiply-add, one packed instruction each.
B200_DEVINL float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
B200_DEVINL float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
        "l"(*reinterpret_cast<unsigned long long*>(&c)));
  return *reinterpret_cast<float2*>(&r);
}

// Statistics of a row of logits relative to a reference m (its running maximum):
// s = sum e^(x - m), w = sum e^(x - m) (x - m). m = -inf: nothing but -inf so far, s = w = 0.
struct LogitStat {
  float m, s, w;
};

B200_DEVINL LogitStat logit_stat_empty() { return LogitStat{-INFINITY, 0.f, 0.f}; }

// Merge in either order. Moving a part from its m to the larger M, with t = m - M <= 0:
// e^(x - M) = e^(x - m) e^t and x - M = (x - m) + t. A part with m = -inf contributes nothing
// (its t would be NaN or -inf, times zero); a NaN in s passes through.
B200_DEVINL LogitStat logit_stat_merge(const LogitStat& a, const LogitStat& b) {
  LogitStat o;
  o.m = fmaxf(a.m, b.m);
  const float ta = a.m == -INFINITY ? 0.f : a.m - o.m, tb = b.m == -INFINITY ? 0.f : b.m - o.m;
  const float ea = expf(ta), eb = expf(tb);
  // where e^t is 0 (t may be -inf) the part is below fp32's reach: s e^t = 0 and so is its w
  const float wa = ea > 0.f ? (a.w + a.s * ta) * ea : 0.f, wb = eb > 0.f ? (b.w + b.s * tb) * eb : 0.f;
  o.s = a.s * ea + b.s * eb;
  o.w = wa + wb;
  return o;
}

struct RowResult {
  float logprob, entropy, lse;
};

// xt: the token's logit; valid: its id is inside the vocabulary.
B200_DEVINL RowResult logit_stat_finish(const LogitStat& st, float xt, bool valid) {
  RowResult r;
  if (st.m == -INFINITY && !isnan(st.s)) {
    r.lse = -INFINITY;
    r.entropy = 0.f;
    r.logprob = -INFINITY;
  } else {
    const float ls = logf(st.s);
    r.lse = st.m + ls;
    r.entropy = fmaxf(ls - st.w / st.s, 0.f);        // (a sum a rounding below 1 has a logarithm below 0)
    r.logprob = fminf((xt - st.m) - ls, 0.f);
  }
  if (isnan(st.s)) r.lse = r.entropy = r.logprob = NAN;
  if (!valid) r.logprob = NAN;
  return r;
}

}  // namespace b200
