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
// once: its sums, and each thread's maximum. A workgroup per row joins the slices' sums in order and finds the alternatives:
// the `top` largest scores lie with threads whose maxima are among the largest, so the maxima (1/32 of the scores' bytes)
// name the few pieces of the row that are read again. Few rows are bound by the two launches' latency. Many are bound by
// memory, and nearly by the vector units (a score costs some ten instructions, an exponential at a quarter of the rate among
// them): 1021 rows of 151936 scores in 57 us, 5.4 TB/s, without alternatives, in 65 with 1 to 32 of them. Alternatives
// looked for slice by slice cost every wave a search of its own: 77 us for 5, 91 for 32.
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

// Eight scores from number `at` on, those past the `n`-th -inf.
__device__ __forceinline__ u32x4_t piece_of(const uint16_t* scores, int at, int n) {
  if (at + 8 <= n) return *reinterpret_cast<const u32x4_any_t*>(scores + at);
  u32x4_t raw;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = at + 2 * i;
    raw[i] = (e < n ? scores[e] : 0xff80u) | (e + 1 < n ? (uint32_t)scores[e + 1] << 16 : 0xff800000u);
  }
  return raw;
}

// Workspace: per (row, slice) the maximum, Z, W and a word of nothing; then, where there are alternatives to find, per row
// the maxima of its slices' threads as bf16.
constexpr int kHead = 4;  // words

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

template <int kCtrl>
__device__ __forceinline__ float dpp_fmax(float v) {
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xF, 0xF, false)));
}
__device__ __forceinline__ float wave_fmax(float v) {
  v = dpp_fmax<0xB1>(v);
  v = dpp_fmax<0x4E>(v);
  v = dpp_fmax<0x141>(v);
  v = dpp_fmax<0x140>(v);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
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

constexpr uint32_t kNegInf = 0x7fu;  // order_of(-inf)

__global__ __launch_bounds__(kThreads) void logprobs_slice_kernel(const uint16_t* __restrict__ logits, int V, int64_t ld,
                                                                  float inv_temp, float* __restrict__ heads,
                                                                  uint16_t* __restrict__ maxima) {
  __shared__ float sums[3][kWaves];
  const int slice = blockIdx.x, wave = wave_id();
  const size_t r = blockIdx.y;
  const int base = slice * kSlice, n = min(kSlice, V - base);
  const uint16_t* src = logits + (int64_t)r * ld + base;
  u32x4_t raw[kPieces];
  if (n == kSlice) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) raw[j] = *reinterpret_cast<const u32x4_any_t*>(src + 8 * (threadIdx.x + j * kThreads));
  } else {  // the row's last slice: what is past it is -inf, which adds nothing
#pragma unroll
    for (int j = 0; j < kPieces; ++j) raw[j] = piece_of(src, 8 * (threadIdx.x + j * kThreads), n);
  }
  float x[kPieces][8];
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[j][2 * i] = __uint_as_float(raw[j][i] << 16);
      x[j][2 * i + 1] = __uint_as_float(raw[j][i] & 0xffff0000u);
    }
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, x[j][e]);
  const size_t at = r * gridDim.x + slice;
  if (maxima) maxima[at * kThreads + threadIdx.x] = (uint16_t)(__float_as_uint(m) >> 16);
  m = wave_fmax(m);  // each wave's sums are relative to its own maximum
  const float mref = m == -INFINITY ? 0.f : m, c = inv_temp * kLog2e;
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
  if ((threadIdx.x & 63) == 0) {
    sums[0][wave] = m;
    sums[1][wave] = z;
    sums[2][wave] = -s;
  }
  __syncthreads();
  if (threadIdx.x) return;
  // The waves' sums, each brought to the slice's maximum; nothing but -inf adds nothing, or NaN where its sum is.
  m = fmaxf(fmaxf(sums[0][0], sums[0][1]), fmaxf(sums[0][2], sums[0][3]));
  float w = 0.f;
  z = 0.f;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    const float mv = sums[0][v], zv = sums[1][v];
    const float f = mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mv - m) * c);
    z += mv == -INFINITY ? zv : zv * f;
    w += f == 0.f ? 0.f : fmaf(zv, m - mv, sums[2][v]) * f;
  }
  *reinterpret_cast<f32x4_t*>(heads + at * kHead) = f32x4_t{m, z, w, 0.f};
}

// One workgroup per row. Lane j of each wave holds slice j's sums; the threads' maxima are spread over its threads. A bound
// that at least `top` maxima reach comes from its threads' own maxima: every wave has ceil(top / 4) threads that reach the
// least of the waves' values for that count; for one or two, the greatest of the waves' values for the whole count lies
// nearer. The threads' parts of the row whose maximum reaches it are read again, and the scores that reach it ranked by
// counting those above.
constexpr int kChunks = 256;                                  // threads' parts that are read again
constexpr int kScores = 1024;                                 // scores that a list holds; at least 32 (kMaxTop - 1)
constexpr int kRanked = 256;                                  // and that are ranked if there is another way

// kLoads: 16-byte pieces of maxima per thread, 8 slices' each, which stay in registers (46, 58 and 107 in all for 1, 4 and 8
// of them): 4096 rows of 32768 scores, 5 alternatives, 65 us with 8, 56 with 1.
template <int kLoads>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(const uint16_t* __restrict__ logits, int64_t ld, int V,
                                                                 const int32_t* __restrict__ tokens, float inv_temp, int top,
                                                                 int slices, const float* __restrict__ heads,
                                                                 const uint16_t* __restrict__ maxima,
                                                                 float* __restrict__ logprob, float* __restrict__ entropy,
                                                                 int32_t* __restrict__ ids, float* __restrict__ top_logprob) {
  __shared__ uint32_t chunks[kChunks], red[kWaves], counts[2], first;
  __shared__ __attribute__((aligned(16))) uint64_t scores[kScores];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const size_t r = blockIdx.x;
  const uint16_t* row = logits + (int64_t)r * ld;
  const bool have = lane < slices;
  const f32x4_t mine = *reinterpret_cast<const f32x4_t*>(heads + (r * slices + min(lane, slices - 1)) * kHead);
  const int token = tokens[r];
  const float x = token >= 0 && token < V ? bf16_bits_to_f32(row[token]) : -INFINITY;
  // Piece number i of the row's maxima, eight threads' of slice i / 32: four waves in turn, so that few pieces are shared too.
  const int pieces = slices * (kThreads / 8);
  u32x4_t mx[kLoads];
  float best = -INFINITY;
  if (top) {
    if (threadIdx.x < 2) counts[threadIdx.x] = 0;
    const u32x4_t* src = reinterpret_cast<const u32x4_t*>(maxima + r * slices * kThreads);
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      mx[k] = u32x4_t{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
      if (kThreads * k < pieces) {
        const int i = kThreads * k + 4 * lane + wave;
        if (i < pieces) mx[k] = src[i];
      }
    }
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      if (kThreads * k < pieces)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          best = fmaxf(best, fmaxf(__uint_as_float(mx[k][e] << 16), __uint_as_float(mx[k][e] & 0xffff0000u)));
  }
  const float ms = have ? mine[0] : -INFINITY;
  float z = have ? mine[1] : 0.f, w = have ? mine[2] : 0.f;
  const float m = wave_fmax(ms);
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
  auto put = [&](int place, uint32_t order, int index) {
    ids[r * top + place] = index;
    top_logprob[r * top + place] = (value_of(order) - m) * inv_temp - ln_z;
  };
  // The scores of the listed parts (c: thread c % 256 of slice c / 256) that reach `least`, listed; 16 bytes a thread.
  auto gather = [&](int n, uint32_t least) {
    for (int i = threadIdx.x; i < 4 * n; i += kThreads) {
      const int c = chunks[i >> 2], at = c / kThreads * kSlice + 8 * (c % kThreads + (i & 3) * kThreads);
      const u32x4_t raw = piece_of(row, at, V);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t o = order_of(e & 1 ? raw[e >> 1] >> 16 : raw[e >> 1] & 0xffffu);
        if (o >= least && at + e < V) {
          const uint32_t to = atomicAdd(&counts[1], 1u);
          if (to < kScores) scores[to] = (uint64_t)o << 32 | (0xffffffffu - (at + e));
        }
      }
    }
    __syncthreads();
    const int all = counts[1];
    if (threadIdx.x < 3 && all + threadIdx.x < kScores) scores[all + threadIdx.x] = 0;  // to whole fours
    __syncthreads();
    return all;
  };
  // A listed score's place is the number of those above it; no two are equal.
  auto rank = [&](int n) {
    for (int c = threadIdx.x; c < n; c += kThreads) {
      const uint64_t k = scores[c];
      int place = 0;
      for (int i = 0; i < n; i += 4)
#pragma unroll
        for (int e = 0; e < 4; ++e) place += scores[i + e] > k ? 1 : 0;
      if (place < top) put(place, (uint32_t)(k >> 32), (int)(0xffffffffu - (uint32_t)k));
    }
  };
  const int need = top <= 2 ? top : (top + kWaves - 1) / kWaves;
  const uint32_t own = order_of(__float_as_uint(best) >> 16);
  uint32_t least = reached_by(own, wave_max(own), need);
  if (lane == 0) red[wave] = least;
  __syncthreads();
  least = red[0];
#pragma unroll
  for (int v = 1; v < kWaves; ++v) least = top <= 2 ? max(least, red[v]) : min(least, red[v]);
  // The threads' parts whose maximum reaches `at_least`, listed.
  auto list_chunks = [&](uint32_t at_least) {
    const float bound = value_of(at_least);
    if (best >= bound)
#pragma unroll
      for (int k = 0; k < kLoads; ++k)
        if (kThreads * k < pieces)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (__uint_as_float(e & 1 ? mx[k][e >> 1] & 0xffff0000u : mx[k][e >> 1] << 16) >= bound) {
              const uint32_t to = atomicAdd(&counts[0], 1u);
              if (to < kChunks) chunks[to] = 8 * (kThreads * k + 4 * lane + wave) + e;
            }
    __syncthreads();
    return (int)counts[0];
  };
  if (least > kNegInf) {
    const int n = list_chunks(least);
    if (n <= kChunks) {
      const int all = gather(n, least);
      if (all <= kRanked) {
        rank(all);
        return;
      }
    }
  }
  // Too many equal scores to list, or too few that are not -inf (1021 rows of 151936 with 3 scores each that are: 81 us
  // for 5 alternatives, all scores equal 83, some thousand equal ones last 85): `least` becomes the top-th largest of the maxima,
  // bit by bit. Fewer than `top` lie above it, whose scores fit the lists.
  least = 0;
#pragma unroll 1
  for (int bit = 15; bit >= 0; --bit) {
    const uint32_t next = least | 1u << bit;
    int reach = 0;
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t o = order_of(e & 1 ? mx[k][e >> 1] >> 16 : mx[k][e >> 1] & 0xffffu);
        reach += __popcll(ballot(o >= next));
      }
    __syncthreads();
    if (lane == 0) red[wave] = reach;
    __syncthreads();
    least = (int)(red[0] + red[1] + red[2] + red[3]) >= top ? next : least;
  }
  __syncthreads();
  if (threadIdx.x < 2) counts[threadIdx.x] = 0;
  if (threadIdx.x == 0) first = slices;
  __syncthreads();
  const float bound = value_of(least);
  uint32_t before = 0;  // slices from this thread's first such part on
#pragma unroll
  for (int k = kLoads - 1; k >= 0; --k) {
    float most = __uint_as_float(mx[k][0] << 16);
#pragma unroll
    for (int e = 1; e < 8; ++e) most = fmaxf(most, __uint_as_float(e & 1 ? mx[k][e >> 1] & 0xffff0000u : mx[k][e >> 1] << 16));
    const int slice = (kThreads * k + 4 * lane + wave) / (kThreads / 8);
    if (most >= bound && slice < slices) before = slices - slice;
  }
  before = wave_max(before);
  if (lane == 0) atomicMin(&first, slices - before);
  const int above = gather(list_chunks(least + 1), least + 1);
  rank(above);
  // Then those equal to it, from the first slice that has one, and last the NaN ones, by their indices.
  int placed = above;
  for (uint32_t target = least;; target = 1u) {
#pragma unroll 1
    for (int base = target == least ? (int)first * kSlice : 0; base < V && placed < top; base += 8 * kThreads) {
      const int at = base + 8 * threadIdx.x;
      const u32x4_t raw = piece_of(row, at, V);
      uint32_t equal = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t o = order_of(e & 1 ? raw[e >> 1] >> 16 : raw[e >> 1] & 0xffffu);
        equal |= (o == target && at + e < V ? 1u : 0u) << e;
      }
      const int own_count = __popc(equal);
      int upto = own_count;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(upto, o, 64);
        upto += lane >= o ? v : 0;
      }
      __syncthreads();
      if (lane == 63) red[wave] = upto;
      __syncthreads();
      int place = placed + upto - own_count;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        place += v < wave ? (int)red[v] : 0;
        placed += red[v];
      }
      for (; equal && place < top; equal &= equal - 1, ++place) put(place, target, at + __builtin_ctz(equal));
    }
    if (target == 1u || placed >= top) return;
  }
}

}  // namespace

extern "C" size_t skinny_token_logprobs_workspace_bytes(int rows, int V, int top) {
  if (rows < 1 || V < 1 || V > kSlice * kMaxSlices || top < 0 || top > kMaxTop) return 0;
  return (size_t)rows * ((V + kSlice - 1) / kSlice) * (kHead * sizeof(float) + (top ? kThreads * sizeof(uint16_t) : 0));
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
  SKINNY_CHECK_ARG(skinny_aligned(logits, 2) && skinny_aligned(tokens, 4) && skinny_aligned(workspace, 16),
                   "token_logprobs: misaligned buffer");
  const size_t need = skinny_token_logprobs_workspace_bytes(rows, V, top);
  SKINNY_CHECK_ARG(workspace_bytes >= need, "token_logprobs: workspace of %zu bytes, needs %zu", workspace_bytes, need);
  const int slices = (V + kSlice - 1) / kSlice;
  const hipStream_t s = (hipStream_t)stream;
  float* heads = static_cast<float*>(workspace);
  uint16_t* maxima = top ? reinterpret_cast<uint16_t*>(heads + (size_t)rows * slices * kHead) : nullptr;
  hipLaunchKernelGGL(logprobs_slice_kernel, dim3(slices, rows), dim3(kThreads), 0, s, logits, V, ld, inv_temp, heads, maxima);
  if (const int rc = skinny_check_launch("token_logprobs")) return rc;
  auto join = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(rows), dim3(top ? kThreads : 64), 0, s, logits, ld, V, tokens, inv_temp, top, slices, heads,
                       maxima, logprob, entropy, ids, top_logprob);
  };
  if (slices <= 8) join(logprobs_join_kernel<1>);
  else if (slices <= 32) join(logprobs_join_kernel<4>);
  else join(logprobs_join_kernel<8>);
  return skinny_check_launch("token_logprobs join");
}
