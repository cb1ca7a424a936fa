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
// once: its maximum, its sums, and its candidates, the scores that reach a bound which `top` of them are known to reach; a
// workgroup per row joins the slices, sums in order and keys by the same kind of bound. Few rows are bound by the two
// launches' latency. Many are bound by memory and the vector units alike (a score costs some ten instructions, an
// exponential at a quarter of the rate among them): 1021 rows of 151936 scores in 58 us, 5.4 TB/s, without alternatives,
// 81 with 5, 93 with 32. Loads for the next slice kept in flight took registers that the other waves need: 69 and 97 us.
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

// Workspace: per (row, slice) the maximum, Z, W, a word of nothing, then keys (order << 16 | 0xffff - index in the slice) in
// any order, the slice's `top` largest among them, and zeros.
__host__ __device__ constexpr int part_keys(int top) { return top ? 2 * top + 8 : 0; }
__host__ __device__ constexpr int part_words(int top) { return 4 + part_keys(top); }

// The lanes for which a condition holds, straight from its compare.
__device__ __forceinline__ uint64_t ballot(bool b) { return __builtin_amdgcn_ballot_w64(b); }

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

// The largest value that `need` lanes reach (0: not so many have one), their largest being `largest`.
__device__ __forceinline__ uint32_t reached_by(uint32_t v, uint32_t largest, int need) {
  if (need <= 4) {  // from the top
    uint32_t least = largest;
    while (least && __popcll(ballot(v >= least)) < need) least = wave_max(v < least ? v : 0u);
    return least;
  }
  uint32_t least = 0;  // bit by bit
#pragma unroll
  for (int bit = 15; bit >= 0; --bit) {
    const uint32_t next = least | 1u << bit;
    least = __popcll(ballot(v >= next)) >= need ? next : least;
  }
  return least;
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
  u32x4_t raw[kPieces];
  if (n == kSlice) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) raw[j] = *reinterpret_cast<const u32x4_any_t*>(src + 8 * (threadIdx.x + j * kThreads));
  } else {  // the row's last slice: what is past it is -inf, which adds nothing
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int e0 = 8 * (threadIdx.x + j * kThreads);
      raw[j] = u32x4_t{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
      if (e0 + 8 <= n) {
        raw[j] = *reinterpret_cast<const u32x4_any_t*>(src + e0);
      } else if (e0 < n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = e0 + 2 * i;
          raw[j][i] = (e < n ? src[e] : 0xff80u) | (e + 1 < n ? (uint32_t)src[e + 1] << 16 : 0xff800000u);
        }
      }
    }
  }
  float x[kPieces][8];
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[j][2 * i] = __uint_as_float(raw[j][i] << 16);
      x[j][2 * i + 1] = __uint_as_float(raw[j][i] & 0xffff0000u);
    }
  float m = -INFINITY, most[kPieces];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    most[j] = x[j][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) most[j] = fmaxf(most[j], x[j][e]);
    m = fmaxf(m, most[j]);
  }
  // The slice's maximum, and a value that at least `top` of its scores reach, from the threads' maxima: every wave has
  // ceil(top / 4) that reach the least of the waves' values for that count; for one or two, the greatest of the waves'
  // values for the whole count lies nearer.
  const uint32_t mine = order_of(__float_as_uint(m) >> 16);
  const int need = top <= 2 ? top : (top + kWaves - 1) / kWaves;
  const uint32_t largest = wave_max(mine);
  const uint32_t least0 = top ? reached_by(mine, largest, need) : 0u;
  if (lane == 0) {
    red[0][wave] = largest;
    red[1][wave] = least0;
  }
  __syncthreads();
  uint32_t om = red[0][0], least = red[1][0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    om = max(om, red[0][w]);
    least = top <= 2 ? max(least, red[1][w]) : min(least, red[1][w]);
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
    for (int j = 0; j < kPieces; ++j) {
      if (!ballot(most[j] >= bound)) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint64_t who = ballot(x[j][e] >= bound);
        if (who) {
          const int at = found + __popcll(who & ((1ull << lane) - 1));
          if ((who >> lane & 1) && at < kList)
            list[wave][at] = order_of(__float_as_uint(x[j][e]) >> 16) << 16 | (0xffffu - 8 * (threadIdx.x + j * kThreads) - e);
          found += __popcll(who);
        }
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
  int all = 0, before = 0;
  bool fits = true;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? (int)count[w] : 0;
    all += count[w];
    fits &= count[w] <= kList;
  }
  fits &= all >= top;
  const bool listed = fits && all <= part_keys(top);
  for (int i = (listed ? all : top) + threadIdx.x; i < part_keys(top); i += kThreads) part[4 + i] = 0;
  if (listed) {
    if (lane < (int)count[wave]) part[4 + before + lane] = list[wave][lane];
    return;
  }
  if (fits) {
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

// One workgroup per row. Lane j of each wave holds slice j's sums; the slices' keys are spread over the threads, and the
// row's largest are found as a slice's are: by a bound from the threads' maxima, then by counting those above.
constexpr int kJoinKeys = kMaxSlices * part_keys(kMaxTop);
constexpr int kJoinList = 512;

__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(const uint16_t* __restrict__ logits, int64_t ld, int V,
                                                                 const int32_t* __restrict__ tokens, float inv_temp, int top,
                                                                 int slices, const uint32_t* __restrict__ parts,
                                                                 float* __restrict__ logprob, float* __restrict__ entropy,
                                                                 int32_t* __restrict__ ids, float* __restrict__ top_logprob) {
  __shared__ uint32_t keys[kJoinKeys], red[kWaves], count;
  __shared__ __attribute__((aligned(16))) uint64_t list[kJoinList + 1];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const size_t r = blockIdx.x;
  const int words = part_words(top), per = part_keys(top);
  const uint32_t* rows = parts + r * slices * words;
  const uint32_t* mine = rows + min(lane, slices - 1) * words;
  const bool have = lane < slices;
  const int token = tokens[r];
  const float x = token >= 0 && token < V ? bf16_bits_to_f32(logits[(int64_t)r * ld + token]) : -INFINITY;
  const float ms = have ? __uint_as_float(mine[0]) : -INFINITY;
  float z = have ? __uint_as_float(mine[1]) : 0.f, w = have ? __uint_as_float(mine[2]) : 0.f;
  // A thread's keys: number i of the row is number i % per of slice i / per.
  const int total = slices * per;
  uint32_t best = 0;
  if (top) {
    if (threadIdx.x == 0) count = 0;
    const int ds = kThreads / per, dq = kThreads % per;
    int s = threadIdx.x / per, q = threadIdx.x % per;
    for (int i = threadIdx.x; i < total; i += kThreads) {
      const uint32_t key = rows[s * words + 4 + q];
      keys[i] = key;
      best = max(best, key >> 16);
      s += ds;
      q += dq;
      if (q >= per) {
        q -= per;
        ++s;
      }
    }
  }
  float m = ms;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ms - m) * inv_temp * kLog2e);
  if (ms != -INFINITY) w = fmaf(z, m - ms, w);
  z = wave_sum(ms == -INFINITY ? z : z * f);
  w = wave_sum(f == 0.f ? 0.f : w * f);
  const float ln_z = logf(z);
  if (threadIdx.x == 0) {
    logprob[r] = (x - m) * inv_temp - ln_z;
    entropy[r] = ln_z + w / z * inv_temp;
  }
  if (!top) return;
  const int need = top <= 2 ? top : (top + kWaves - 1) / kWaves;
  uint32_t least = reached_by(best, wave_max(best), need);
  if (lane == 0) red[wave] = least;
  __syncthreads();
  least = red[0];
#pragma unroll
  for (int v = 1; v < kWaves; ++v) least = top <= 2 ? max(least, red[v]) : min(least, red[v]);
  // A key of the row orders by its score, then by the lower index.
  auto whole = [&](int i) {
    const uint32_t key = keys[i];
    return (uint64_t)(key >> 16) << 32 | (0xffffffffu - (i / per * kSlice + (0xffffu - (key & 0xffffu))));
  };
  auto put = [&](int place, uint64_t k) {
    ids[r * top + place] = (int)(0xffffffffu - (uint32_t)k);
    top_logprob[r * top + place] = (value_of((uint32_t)(k >> 32)) - m) * inv_temp - ln_z;
  };
  if (best >= max(least, 1u))
    for (int i = threadIdx.x; i < total; i += kThreads)
      if (keys[i] >> 16 >= max(least, 1u)) {
        const uint32_t at = atomicAdd(&count, 1u);
        if (at < kJoinList) list[at] = whole(i);
      }
  __syncthreads();
  const int n = count;
  if (n <= kJoinList) {
    for (int c = threadIdx.x; c < n; c += kThreads) {
      const uint64_t k = list[c];
      int place = 0;
      for (int i = 0; i < n; ++i) place += list[i] > k ? 1 : 0;
      if (place < top) put(place, k);
    }
    return;
  }
  // Very many equal scores: one after the other.
  uint64_t prev = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t next = 0;
    for (int i = threadIdx.x; i < total; i += kThreads) {
      const uint64_t v = whole(i);
      if (keys[i] && v < prev && v > next) next = v;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t v = __shfl_xor((unsigned long long)next, o, 64);
      next = v > next ? v : next;
    }
    __syncthreads();
    if (lane == 0) list[wave] = next;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kWaves; ++v) next = list[v] > next ? list[v] : next;
    if (threadIdx.x == 0) put(k, next);
    prev = next;
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
  SKINNY_CHECK_ARG(inv_temp > 0.f && inv_temp <= 1.0e38f, "token_logprobs: bad temperature");
  SKINNY_CHECK_ARG(skinny_aligned(logits, 2) && skinny_aligned(tokens, 4) && skinny_aligned(workspace, 4),
                   "token_logprobs: misaligned buffer");
  const size_t need = skinny_token_logprobs_workspace_bytes(rows, V, top);
  SKINNY_CHECK_ARG(workspace_bytes >= need, "token_logprobs: workspace of %zu bytes, needs %zu", workspace_bytes, need);
  const int slices = (V + kSlice - 1) / kSlice;
  const hipStream_t s = (hipStream_t)stream;
  uint32_t* parts = static_cast<uint32_t*>(workspace);
  hipLaunchKernelGGL(logprobs_slice_kernel, dim3(slices, rows), dim3(kThreads), 0, s, logits, V, ld, inv_temp, top, parts);
  if (const int rc = skinny_check_launch("token_logprobs")) return rc;
  hipLaunchKernelGGL(logprobs_join_kernel, dim3(rows), dim3(top ? kThreads : 64), 0, s, logits, ld, V, tokens, inv_temp, top, slices, parts,
                     logprob, entropy, ids, top_logprob);
  return skinny_check_launch("token_logprobs join");
}
