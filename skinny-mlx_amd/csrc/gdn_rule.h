// The gated delta rule's token update and what its kernels share: one sequence's (gdn.hip) and several sequences'
// (gdn_batch.hip).
#pragma once

#include "common.h"

namespace {

constexpr int kDk = 128, kDv = 128;
constexpr int kCols = 8;   // value columns per workgroup (H x 16 workgroups)
constexpr int kPart = 16;  // lanes per column (8 key dims each)

__device__ __forceinline__ float sum16(float v) { return row16_sum(v); }

__device__ __forceinline__ float softplus(float x) { return x > 20.f ? x : log1pf(expf(x)); }

constexpr int kTokBlock = 16;  // tokens staged per pass (and the most that a draft tree may hold)

// One token of the gated delta rule for the 8 key dims a lane holds of one value column (the
// column's 16 lanes together hold all 128): S <- decay S + k delta with delta = beta (v - k.(decay
// S)), then y = q.S. k.S is formed on the undecayed state and scaled once (decay (k.S)), in four
// partial sums, and so is q.S: short dependency chains, since the tokens run one after another.
// Returns y (the same in all 16 lanes of the column).
__device__ __forceinline__ float gdn_token(float (&s)[8], const float (&kh)[8], const float (&qh)[8], float v,
                                           float decay, float beta) {
  float a0 = s[0] * kh[0], a1 = s[1] * kh[1], a2 = s[2] * kh[2], a3 = s[3] * kh[3];
  a0 = fmaf(s[4], kh[4], a0);
  a1 = fmaf(s[5], kh[5], a1);
  a2 = fmaf(s[6], kh[6], a2);
  a3 = fmaf(s[7], kh[7], a3);
  const float delta = beta * (v - decay * sum16((a0 + a1) + (a2 + a3)));
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = fmaf(kh[e], delta, s[e] * decay);
  float b0 = s[0] * qh[0], b1 = s[1] * qh[1], b2 = s[2] * qh[2], b3 = s[3] * qh[3];
  b0 = fmaf(s[4], qh[4], b0);
  b1 = fmaf(s[5], qh[5], b1);
  b2 = fmaf(s[6], qh[6], b2);
  b3 = fmaf(s[7], qh[7], b3);
  return sum16((b0 + b1) + (b2 + b3));
}

}  // namespace
