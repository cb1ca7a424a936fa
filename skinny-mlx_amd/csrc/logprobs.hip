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
// once: its maximum, its sums, and its largest scores, which are picked out by a bound that `top` of them reach; a wave
// per row joins the slices in order. Many rows are bound by memory and the vector units alike: a score costs about ten
// instructions, one of them an exponential at a quarter of the rate.
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

// The largest value over the wave, in every lane.
template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = dpp_max<0xB1>(v);   // quad_perm [1,0,3,2]
  v = dpp_max<0x4E>(v);   // quad_perm [2,3,0,1]
  v = dpp_max<0x141>(v);  // row_half_mirror
  v = dpp_max<0x140>(v);  // row_mirror
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(b[0], b[1]);
}

constexpr int kWaves = kThreads / 64;
constexpr int kList = 64;  // candidates that a wave may have; a slice with more (many equal scores) goes the long way
constexpr uint32_t kNegInf = 0x7fu;  // order_of(-inf)

__global__ __launch_bounds__(kThreads) void logprobs_slice_kernel(const uint16_t* __restrict__ logits, int V, int64_t ld,
                                                                  float inv_temp, int top, uint32_t* __restrict__ parts) {
  __shared__ uint32_t red[2][kWaves], count[kWaves];
  __shared__ float sums[2][kWaves];
  __shared__ __attribute__((aligned(16))) uint32_t list[kWaves][kList + 4];
  const int slice = blockIdx.x, lane = threadIdx.x & 63, wave = wave_id();
  const size_t r = blockIdx.y;
  const uint16_t* row = logits + (int64_t)r * ld;
  const int base = slice * kSlice, n = min(kSlice, V - base);
  const uint16_t* src = row + base;
  float x[kPieces][8];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int e0 = 8 * (threadIdx.x + j * kThreads);
    u32x4_t w;
    if (e0 + 8 <= n) {
      w = *reinterpret_cast<const u32x4_any_t*>(src + e0);
    } else {  // the row's last scores; what is past them is -inf, which adds nothing
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + 2 * i;
        w[i] = (e < n ? src[e] : 0xff80u) | (e + 1 < n ? (uint32_t)src[e + 1] << 16 : 0xff800000u);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[j][2 * i] = __uint_as_float(w[i] << 16);
      x[j][2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, x[j][e]);
  // The slice's maximum, and a value that at least `top` of its scores reach: the largest for which that many threads of
  // some wave have one.
  const uint32_t mine = order_of(__float_as_uint(m) >> 16);
  uint32_t least = 0;
  if (top) {
#pragma unroll
    for (int bit = 15; bit >= 0; --bit) {
      const uint32_t next = least | 1u << bit;
      least = __popcll(__ballot(mine >= next)) >= top ? next : least;
    }
  }
  const uint32_t largest = wave_max(mine);
  if (lane == 0) {
    red[0][wave] = largest;
    red[1][wave] = least;
  }
  __syncthreads();
  uint32_t om = red[0][0];
  least = red[1][0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    om = max(om, red[0][w]);
    least = max(least, red[1][w]);
  }
  m = value_of(om);
  const float mref = om <= kNegInf ? 0.f : m, c = inv_temp * kLog2e;
  // Banned scores and those far below lose their sign of infinity here, for 0 * inf is no number.
  float z = 0.f, s = 0.f;
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = x[j][e] - mref;
      const float p = __builtin_amdgcn_exp2f(d * c);
      z += p;
      s = fmaf(p, fmaxf(d, -3e38f), s);
    }
  z = wave_sum(z);
  s = wave_sum(s);
  // Candidates: the scores that reach `least`, each wave's in a list of its own.
  const float bound = value_of(least);
  int found = 0;
  if (top && least > kNegInf) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint64_t who = __ballot(x[j][e] >= bound);
        if (who) {
          const int at = found + __popcll(who & ((1ull << lane) - 1));
          if ((who >> lane & 1) && at < kList)
            list[wave][at] = order_of(__float_as_uint(x[j][e]) >> 16) << 16 | (0xffffu - 8 * (threadIdx.x + j * kThreads) - e);
          found += __popcll(who);
        }
      }
    if (lane < 4) list[wave][min(found, kList) + lane] = 0;  // to a whole piece
  }
  if (lane == 0) {
    sums[0][wave] = z;
    sums[1][wave] = s;
    count[wave] = found;
  }
  __syncthreads();
  uint32_t* part = parts + (r * gridDim.x + slice) * part_words(top);
  if (threadIdx.x == 0) {
    float zt = 0.f, st = 0.f;
    for (int w = 0; w < kWaves; ++w) {
      zt += sums[0][w];
      st += sums[1][w];
    }
    part[0] = __float_as_uint(m);
    part[1] = __float_as_uint(zt);
    part[2] = __float_as_uint(-st);
  }
  if (!top) return;
  int all = 0;
  bool fits = true;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    all += count[w];
    fits &= count[w] <= kList;
  }
  if (fits && all >= top) {
    // Keys are all different: a candidate's place is the number of those above it.
    if (lane >= (int)count[wave]) return;
    const uint32_t key = list[wave][lane];
    int place = 0;
    for (int w = 0; w < kWaves; ++w)
      for (int i = 0; i < (int)count[w]; i += 4) {
        const u32x4_t k4 = *reinterpret_cast<const u32x4_t*>(&list[w][i]);
#pragma unroll
        for (int q = 0; q < 4; ++q) place += k4[q] > key ? 1 : 0;
      }
    if (place < top) part[4 + place] = key;
    return;
  }
  // The long way: the largest keys one after the other.
  uint32_t prev = 0xffffffffu;
  for (int k = 0; k < top; ++k) {
    uint32_t best = 0;
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = 8 * (threadIdx.x + j * kThreads) + e;
        const uint32_t key = (order_of(__float_as_uint(x[j][e]) >> 16) << 16) | (0xffffu - (uint32_t)i);
        if (i < n && key < prev) best = max(best, key);
      }
    best = wave_max(best);
    __syncthreads();
    if (lane == 0) red[0][wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) best = max(best, red[0][w]);
    if (threadIdx.x == 0) part[4 + k] = best;
    prev = best;
  }
}

// One wave per row; lane j holds slice j.
__global__ __launch_bounds__(64) void logprobs_join_kernel(const uint16_t* __restrict__ logits, int64_t ld, int V,
                                                           const int32_t* __restrict__ tokens, float inv_temp, int top,
                                                           int slices, const uint32_t* __restrict__ parts,
                                                           float* __restrict__ logprob, float* __restrict__ entropy,
                                                           int32_t* __restrict__ ids, float* __restrict__ top_logprob) {
  __shared__ uint32_t keys[kMaxSlices * kMaxTop];
  const int lane = threadIdx.x;
  const size_t r = blockIdx.x;
  const uint32_t* rows = parts + r * slices * part_words(top);
  const uint32_t* mine = rows + min(lane, slices - 1) * part_words(top);
  const bool have = lane < slices;
  const int token = tokens[r];
  const float x = token >= 0 && token < V ? bf16_bits_to_f32(logits[(int64_t)r * ld + token]) : -INFINITY;
  const float ms = have ? __uint_as_float(mine[0]) : -INFINITY;
  float z = have ? __uint_as_float(mine[1]) : 0.f, w = have ? __uint_as_float(mine[2]) : 0.f;
  for (int i = lane; i < slices * top; i += 64) keys[i] = rows[i / top * part_words(top) + 4 + i % top];
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
  // The slices' keys are in order: the next of the row is at the head of one of them.
  lds_barrier();
  int head = 0;
  for (int k = 0; k < top; ++k) {
    const uint32_t key = have && head < top ? keys[lane * top + head] : 0u;
    const uint32_t order = wave_max(key >> 16);
    const uint64_t who = __ballot(key != 0u && (key >> 16) == order);  // the first slice has the lower indices
    if (lane == __ffsll((unsigned long long)who) - 1) {
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
