// Log-probabilities of given tokens, the entropy of each row's distribution, and its most probable tokens, from
// a head's bf16 scores.
//
// No reference counterpart: the reference reports tokens only (skinny_mlx/spec.py:98-156). The distribution is the
// one that sampling draws from, softmax(row / T) (csrc/sample.hip).
//
// With m the row's maximum, e = exp((x - m) / T), Z = sum e and W = sum e (m - x), all in fp32:
//   log p(token) = (x[token] - m) / T - ln Z,   entropy = ln Z + W / (Z T)
// (every term of W is positive, so nothing cancels). Alternatives are the largest scores, ties by the lower index.
//
// A row is cut into slices of 8192 scores at fixed places. A workgroup holds a slice in registers, so that it is read
// once: its maximum, then its sums, then its largest scores; a wave per row joins the slices in order.
#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kPieces = 4;                          // 16-byte pieces per thread
constexpr int kSlice = kThreads * kPieces * 8;      // scores per slice
constexpr int kMaxSlices = 64;                      // one lane of the joining wave each
constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.4426950408889634f;

// A 16-byte load of scores at any even address: rows of an odd vocabulary lie off the 16-byte grid.
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));

// A score as an unsigned integer that orders as the scores do: NaN lowest (1), then -inf; -0 as +0. 0 is no score.
__device__ __forceinline__ uint32_t order_of(uint32_t bits) {
  if ((bits & 0x7fffu) > 0x7f80u) return 1u;
  if (bits == 0x8000u) bits = 0u;
  return (bits & 0x8000u) ? (~bits & 0xffffu) : (bits | 0x8000u);
}

__device__ __forceinline__ float value_of(uint32_t order) {
  if (order <= 1u) return __builtin_nanf("");
  return bf16_bits_to_f32((order & 0x8000u) ? (order & 0x7fffu) : (~order & 0xffffu));
}

// Workspace: per (row, slice) the maximum, Z and W, then `top` keys (order << 16 | 0xffff - index in the slice),
// decreasing, 0 where the slice has fewer scores.
__host__ __device__ constexpr int part_words(int top) { return 4 + top; }

__global__ __launch_bounds__(kThreads) void logprobs_slice_kernel(const uint16_t* __restrict__ logits, int V, int64_t ld,
                                                                  float inv_temp, int top, uint32_t* __restrict__ parts) {
  __shared__ float red[3][kThreads / 64];
  __shared__ uint32_t best[kThreads / 64];
  const int slice = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const size_t r = blockIdx.y;
  const uint16_t* row = logits + (int64_t)r * ld;
  const int base = slice * kSlice, n = min(kSlice, V - base);
  const uint16_t* src = row + base;
  uint32_t x[kPieces][4];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int e0 = 8 * (threadIdx.x + j * kThreads);
    if (e0 + 8 <= n) {
      const u32x4_any_t v = *reinterpret_cast<const u32x4_any_t*>(src + e0);
#pragma unroll
      for (int w = 0; w < 4; ++w) x[j][w] = v[w];
    } else {  // the row's last scores; what is past them is -inf, which adds nothing
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int e = e0 + 2 * w;
        x[j][w] = (e < n ? src[e] : 0xff80u) | (e + 1 < n ? (uint32_t)src[e + 1] << 16 : 0xff800000u);
      }
    }
  }
  auto at = [&](int j, int e) { return bf16_bits_to_f32((e & 1) ? x[j][e >> 1] >> 16 : x[j][e >> 1] & 0xffffu); };
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, at(j, e));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) m = fmaxf(m, red[0][w]);
  const float mref = m == -INFINITY ? 0.f : m, c = inv_temp * kLog2e;
  float z = 0.f, s = 0.f;
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = at(j, e) - mref;
      const float p = __builtin_amdgcn_exp2f(d * c);
      z += p;
      if (p != 0.f) s = fmaf(p, -d, s);  // 0 * inf of a banned score is nothing
    }
  z = wave_sum(z);
  s = wave_sum(s);
  if (lane == 0) {
    red[1][wave] = z;
    red[2][wave] = s;
  }
  __syncthreads();
  uint32_t* part = parts + (r * gridDim.x + slice) * part_words(top);
  if (threadIdx.x == 0) {
    float zt = 0.f, st = 0.f;
    for (int w = 0; w < kThreads / 64; ++w) {
      zt += red[1][w];
      st += red[2][w];
    }
    part[0] = __float_as_uint(m);
    part[1] = __float_as_uint(zt);
    part[2] = __float_as_uint(st);
  }
  // The largest keys, one after the other.
  uint32_t prev = 0xffffffffu;
  for (int k = 0; k < top; ++k) {
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = 8 * (threadIdx.x + j * kThreads) + e;
        const uint32_t bits = (e & 1) ? x[j][e >> 1] >> 16 : x[j][e >> 1] & 0xffffu;
        const uint32_t key = (order_of(bits) << 16) | (0xffffu - (uint32_t)i);
        if (i < n && key < prev) mine = max(mine, key);
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine = max(mine, (uint32_t)__shfl_xor((int)mine, o, 64));
    if (lane == 0) best[wave] = mine;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) mine = max(mine, best[w]);
    __syncthreads();
    if (threadIdx.x == 0) part[4 + k] = mine;
    prev = mine;
  }
}

// One wave per row; lane j holds slice j.
__global__ __launch_bounds__(64) void logprobs_join_kernel(const uint16_t* __restrict__ logits, int64_t ld, int V,
                                                           const int32_t* __restrict__ tokens, float inv_temp, int top,
                                                           int slices, const uint32_t* __restrict__ parts,
                                                           float* __restrict__ logprob, float* __restrict__ entropy,
                                                           int32_t* __restrict__ ids, float* __restrict__ top_logprob) {
  const int lane = threadIdx.x;
  const size_t r = blockIdx.x;
  const uint32_t* mine = parts + (r * slices + min(lane, slices - 1)) * part_words(top);
  const bool have = lane < slices;
  const int token = tokens[r];
  const float x = token >= 0 && token < V ? bf16_bits_to_f32(logits[(int64_t)r * ld + token]) : -INFINITY;
  const float ms = have ? __uint_as_float(mine[0]) : -INFINITY;
  float z = have ? __uint_as_float(mine[1]) : 0.f, w = have ? __uint_as_float(mine[2]) : 0.f;
  float m = ms;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ms - m) * inv_temp * kLog2e);
  if (ms != -INFINITY) w = fmaf(z, m - ms, w);
  z = wave_sum(ms == -INFINITY ? z : z * f);
  w = wave_sum(f == 0.f ? 0.f : w * f);
  const float ln_z = logf(z);
  if (lane == 0) {
    logprob[r] = (x - m) * inv_temp - ln_z;
    entropy[r] = ln_z + w / z * inv_temp;
  }
  int head = 0;
  for (int k = 0; k < top; ++k) {
    const uint32_t key = have && head < top ? mine[4 + head] : 0u;
    uint32_t order = key >> 16;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) order = max(order, (uint32_t)__shfl_xor((int)order, o, 64));
    const uint64_t who = __ballot(key != 0u && (key >> 16) == order);  // the first slice has the lower indices
    const int first = __ffsll((unsigned long long)who) - 1;
    if (lane == first) {
      ids[r * top + k] = lane * kSlice + (int)(0xffffu - (key & 0xffffu));
      top_logprob[r * top + k] = (value_of(order) - m) * inv_temp - ln_z;
      ++head;
    }
  }
}

}  // namespace

extern "C" size_t skinny_token_logprobs_workspace_bytes(int rows, int V, int top) {
  if (rows < 1 || V < 1 || V > kSlice * kMaxSlices || top < 0 || top > kMaxTop) return 0;
  return (size_t)rows * ((V + kSlice - 1) / kSlice) * part_words(top) * sizeof(uint32_t);
}

extern "C" int skinny_token_logprobs_bf16(const uint16_t* logits, int rows, int V, int64_t ld, const int32_t* tokens,
                                          float inv_temp, int top, void* workspace, size_t workspace_bytes, float* logprob,
                                          float* entropy, int32_t* ids, float* top_logprob, void* stream) {
  SKINNY_CHECK_ARG(rows >= 1 && rows <= 65535 && V >= 1 && V <= kSlice * kMaxSlices && ld >= V,
                   "token_logprobs: bad shape rows=%d (at most 65535) V=%d (at most %d) ld=%lld", rows, V,
                   kSlice * kMaxSlices, (long long)ld);
  SKINNY_CHECK_ARG(top >= 0 && top <= kMaxTop && top <= V, "token_logprobs: top=%d (at most %d, and V)", top, kMaxTop);
  SKINNY_CHECK_ARG(logits && tokens && workspace && logprob && entropy && (top == 0 || (ids && top_logprob)),
                   "token_logprobs: null pointer");
  SKINNY_CHECK_ARG(inv_temp > 0.f && inv_temp <= 3.0e38f, "token_logprobs: bad temperature");
  SKINNY_CHECK_ARG(skinny_aligned(logits, 2) && skinny_aligned(tokens, 4) && skinny_aligned(workspace, 4),
                   "token_logprobs: misaligned buffer");
  const size_t need = skinny_token_logprobs_workspace_bytes(rows, V, top);
  SKINNY_CHECK_ARG(workspace_bytes >= need, "token_logprobs: workspace of %zu bytes, needs %zu", workspace_bytes, need);
  const int slices = (V + kSlice - 1) / kSlice;
  const hipStream_t s = (hipStream_t)stream;
  uint32_t* parts = static_cast<uint32_t*>(workspace);
  hipLaunchKernelGGL(logprobs_slice_kernel, dim3(slices, rows), dim3(kThreads), 0, s, logits, V, ld, inv_temp, top, parts);
  if (const int rc = skinny_check_launch("token_logprobs")) return rc;
  hipLaunchKernelGGL(logprobs_join_kernel, dim3(rows), dim3(64), 0, s, logits, ld, V, tokens, inv_temp, top, slices, parts,
                     logprob, entropy, ids, top_logprob);
  return skinny_check_launch("token_logprobs join");
}
