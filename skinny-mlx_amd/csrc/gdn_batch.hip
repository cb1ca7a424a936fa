// The Gated-DeltaNet pieces of a step of several sequences, their states in a pool: the batched counterpart of
// gdn.hip's one sequence.
//
// No reference counterpart: the reference decodes one sequence (skinny_mlx/spec.py:98-156). Arithmetic of the mixer as
// hooked at skinny_mlx/rollback.py:16, 39-52 (the short causal conv with SiLU, and the gated delta rule
// S <- g S (I - b k k^T) + b v k^T, y = S q).
//
// Sequence b brings counts[b] of at most T new tokens, rows b*T + t. It begins with the pool's state slots[b] (-1: zeros)
// and leaves the one after its tokens in slots_out[b], so sequences may go on from one state, a shared prefix's, each
// into its own. A state that the call writes is no other sequence's.
#include <type_traits>
#include "gdn_rule.h"

namespace {

struct Pool {
  const int32_t *slots, *slots_out, *counts;  // slots_out null: slots; counts null: T each
  int n_slots;
  int64_t stride;  // elements from state to state
};

// A sequence's state read (-1: zeros) and written, and its tokens. Not `ok`: no such state, or no such count.
struct Run {
  int read, write, count;
  bool ok;
};
typedef const __attribute__((address_space(4))) int32_t* words_t;
__device__ __forceinline__ int word(const int32_t* p, int i) { return ((words_t)(uintptr_t)p)[i]; }
__device__ __forceinline__ Run run_of(const Pool& p, int b, int T) {
  const int read = word(p.slots, b), write = p.slots_out ? word(p.slots_out, b) : read;
  const int count = p.counts ? word(p.counts, b) : T;
  return {read, write, count,
          read >= -1 && read < p.n_slots && (unsigned)write < (unsigned)p.n_slots && (unsigned)count <= (unsigned)T};
}

constexpr uint16_t kNanBits = 0x7fc0;

// ---------------------------------------------------------------------------------------------------------
// The conv: a thread per V channels and block of kTokBlock tokens. A token's taps are input rows, or for the first three
// the state's, so the blocks need nothing of each other; the first one reads the state and writes the one after the call.
// Taps oldest first and the exact exponential and division, as gdn.hip's conv: the same bits. For prompts memory and the vector
// units take about as long: 16 sequences of 1000 tokens, 8192 channels, 121 us (4.3 TB/s) with two channels a thread, 135 with
// four and 150 with eight, whose fewer waves load and compute in step.
constexpr int kConvWidth = 4;

template <int V>
struct Chans {
  uint32_t w[(V + 1) / 2];
  typedef uint32_t words_any_t __attribute__((ext_vector_type((V + 1) / 2), aligned(2)));
  __device__ __forceinline__ void load(const uint16_t* p) {
    if constexpr (V > 1) {
      const words_any_t x = *reinterpret_cast<const words_any_t*>(p);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) w[i] = x[i];
    } else {
      w[0] = *p;
    }
  }
  __device__ __forceinline__ void store(uint16_t* p) const {
    if constexpr (V > 1) {
      words_any_t x;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) x[i] = w[i];
      *reinterpret_cast<words_any_t*>(p) = x;
    } else {
      *p = (uint16_t)w[0];
    }
  }
  __device__ __forceinline__ void fill(uint32_t half) {
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) w[i] = half * 0x10001u;
  }
  __device__ __forceinline__ float value(int e) const { return bf16_bits_to_f32(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu); }
};

// v, which the compiler then keeps: it would form it from its 16 bits again for every product.
__device__ __forceinline__ float kept(float v) {
  asm("" : "+v"(v));
  return v;
}
__device__ __forceinline__ uint32_t two_bf16(float a, float b) {
  typedef __attribute__((ext_vector_type(2))) float two_t;
  typedef __attribute__((ext_vector_type(2))) __bf16 two_bf16_t;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(two_t{a, b}, two_bf16_t));
}

template <int V>
__global__ __launch_bounds__(256) void conv_silu_batch_kernel(Pool pool, const uint16_t* __restrict__ x, int64_t ldx, int T, int C,
                                                              uint16_t* state, const uint16_t* __restrict__ weight,
                                                              uint16_t* __restrict__ out, int64_t ldo) {
  constexpr int H = kConvWidth - 1;
  const int c = ((int)blockIdx.x * (int)blockDim.x + (int)threadIdx.x) * V, t0 = (int)blockIdx.y * kTokBlock, b = blockIdx.z;
  if (c >= C) return;
  const Run r = run_of(pool, b, T);
  const int rows = min(kTokBlock, T - t0), live = r.ok ? min(max(r.count - t0, 0), rows) : 0;
  x += (int64_t)b * T * ldx + c;
  out += ((int64_t)b * T + t0) * ldo + c;
  Chans<V> line[H + kTokBlock];
  if (t0 == 0) {
    if (r.ok) {
      const uint16_t* from = state + r.read * pool.stride + c;
#pragma unroll
      for (int j = 0; j < H; ++j)
        if (r.read >= 0) line[j].load(from + (int64_t)j * C);
        else line[j].fill(0);
    }
  } else if (live) {
#pragma unroll
    for (int j = 0; j < H; ++j) line[j].load(x + (int64_t)(t0 - H + j) * ldx);
  }
  Chans<V> words[kConvWidth];  // channel by channel: tap j of channel e is value e * kConvWidth + j
#pragma unroll
  for (int i = 0; i < kConvWidth; ++i) words[i].load(weight + (size_t)c * kConvWidth + i * V);
#pragma unroll
  for (int i = 0; i < kTokBlock; ++i)
    if (i < live) line[H + i].load(x + (int64_t)(t0 + i) * ldx);
  float taps[kConvWidth][V], seen[kConvWidth][V];  // (seen: of the last four tokens, token i's in i % 4)
#pragma unroll
  for (int e = 0; e < V; ++e) {
#pragma unroll
    for (int j = 0; j < kConvWidth; ++j) taps[j][e] = kept(words[(e * kConvWidth + j) / V].value((e * kConvWidth + j) % V));
#pragma unroll
    for (int j = 0; j < H; ++j) seen[j][e] = line[j].value(e);
  }
#pragma unroll
  for (int i = 0; i < kTokBlock; ++i) {
    if (i >= rows) continue;
    Chans<V> y;
    if (i < live) {
      float one[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        seen[(H + i) % kConvWidth][e] = kept(line[H + i].value(e));
        float acc = 0.f;
#pragma unroll
        for (int j = 0; j < kConvWidth; ++j) acc = fmaf(taps[j][e], seen[(i + j) % kConvWidth][e], acc);
        one[e] = acc / (1.0f + expf(-acc));
      }
      if constexpr (V == 1) y.w[0] = f32_to_bf16_bits(one[0]);
      else
#pragma unroll
        for (int e = 0; e < V / 2; ++e) y.w[e] = two_bf16(one[2 * e], one[2 * e + 1]);
    } else {
      y.fill(r.ok ? 0u : kNanBits);
    }
    y.store(out + i * ldo);
  }
  if (t0 != 0 || !r.ok || (r.count == 0 && r.read == r.write)) return;
  // line[count ..]: rows of the state that are left, then the last tokens'
  uint16_t* to = state + r.write * pool.stride + c;
#pragma unroll
  for (int j = 0; j < H; ++j) {
    Chans<V> v;
    const int at = r.count + j;
    if (at >= H) v.load(x + (int64_t)(at - H) * ldx);
    else
#pragma unroll
      for (int i = 0; i < (V + 1) / 2; ++i) v.w[i] = at == 0 ? line[0].w[i] : at == 1 ? line[1].w[i] : line[2].w[i];
    v.store(to + (int64_t)j * C);
  }
}

// ---------------------------------------------------------------------------------------------------------
// The rule token by token: 16 lanes hold a value column (8 key dims each), a group of lanes NC columns, so a workgroup
// 16 * NC of a head's 128; 16 tokens at most. All of the state's loads are issued at once. The token's update is gdn.hip's, its sums in the
// same order: y and the state have the bits of skinny_gdn_recurrence on each sequence alone. Bound by memory for one token (64
// sequences of 32 heads, 271 MB in 59 us), by the vector units for several.
constexpr int kStepThreads = 256, kStepGroups = kStepThreads / kPart;

template <int NC>
__global__ __launch_bounds__(kStepThreads) void gdn_batch_steps_kernel(Pool pool, const uint16_t* __restrict__ qkv, int64_t ldq,
                                                                       const uint16_t* __restrict__ bcol,
                                                                       const uint16_t* __restrict__ acol, int64_t ldab,
                                                                       const float* __restrict__ A_log,
                                                                       const float* __restrict__ dt_bias, float* state,
                                                                       float* __restrict__ y, int T, int H, int Hk) {
  __shared__ __attribute__((aligned(16))) float qk_lds[kTokBlock][2][kDk];  // normalised
  __shared__ float v_lds[kTokBlock][kStepGroups * NC];
  __shared__ float gate_lds[kTokBlock][2];  // decay, beta
  constexpr int COLS = kStepGroups * NC;
  const int h = blockIdx.x, b = blockIdx.z, tid = threadIdx.x;
  const int g = tid / kPart, p = tid % kPart;
  const int col0 = (int)blockIdx.y * COLS;
  const Run r = run_of(pool, b, T);
  const size_t row0 = (size_t)b * T;
  float* yb = y + (row0 * H + h) * kDv + col0;
  const size_t ystep = (size_t)H * kDv;
  {
    const int first = r.ok ? r.count : 0;
    const float fill = r.ok ? 0.f : __builtin_nanf("");
    for (int i = tid; i < (T - first) * COLS; i += kStepThreads) yb[(first + i / COLS) * ystep + i % COLS] = fill;
  }
  if (!r.ok || (r.count == 0 && r.read == r.write)) return;
  const size_t at = ((size_t)h * kDv + col0 + g * NC) * kDk + p * 8;
  float s[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    f32x4_t lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
    if (r.read >= 0) {
      const float* from = state + r.read * pool.stride + at + c * kDk;
      lo = *reinterpret_cast<const f32x4_t*>(from);
      hi = *reinterpret_cast<const f32x4_t*>(from + 4);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[c][e] = lo[e];
      s[c][4 + e] = hi[e];
    }
  }
  const int hk = h / (H / Hk);
  const float neg_a = -expf(A_log[h]), dtb = dt_bias[h], qscale = rsqrtf((float)kDk);
  if (g < r.count) {  // a lane group per token: its q and k, normalised
    const uint16_t* row = qkv + (int64_t)(row0 + g) * ldq + (size_t)hk * kDk + p * 8;
    const u32x4_t qw = *reinterpret_cast<const u32x4_t*>(row);
    const u32x4_t kw = *reinterpret_cast<const u32x4_t*>(row + (size_t)Hk * kDk);
    float q[8], k[8], qq = 0.f, kk = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q[e] = bf16_bits_to_f32((e & 1) ? (qw[e >> 1] >> 16) : (qw[e >> 1] & 0xffffu));
      k[e] = bf16_bits_to_f32((e & 1) ? (kw[e >> 1] >> 16) : (kw[e >> 1] & 0xffffu));
      qq = fmaf(q[e], q[e], qq);
      kk = fmaf(k[e], k[e], kk);
    }
    const float qn = rsqrtf(sum16(qq) + 1e-6f) * qscale, kn = rsqrtf(sum16(kk) + 1e-6f);
    f32x4_t* qd = reinterpret_cast<f32x4_t*>(&qk_lds[g][0][p * 8]);
    f32x4_t* kd = reinterpret_cast<f32x4_t*>(&qk_lds[g][1][p * 8]);
    qd[0] = f32x4_t{q[0] * qn, q[1] * qn, q[2] * qn, q[3] * qn};
    qd[1] = f32x4_t{q[4] * qn, q[5] * qn, q[6] * qn, q[7] * qn};
    kd[0] = f32x4_t{k[0] * kn, k[1] * kn, k[2] * kn, k[3] * kn};
    kd[1] = f32x4_t{k[4] * kn, k[5] * kn, k[6] * kn, k[7] * kn};
    if (p < 2) {
      const float x = bf16_bits_to_f32((p ? bcol : acol)[(int64_t)(row0 + g) * ldab + h]);
      gate_lds[g][p] = p ? 1.0f / (1.0f + expf(-x)) : expf(neg_a * softplus(x + dtb));
    }
  }
  for (int i = tid; i < r.count * COLS; i += kStepThreads)
    v_lds[i / COLS][i % COLS] =
        bf16_bits_to_f32(qkv[(int64_t)(row0 + i / COLS) * ldq + (size_t)2 * Hk * kDk + (size_t)h * kDv + col0 + i % COLS]);
  __syncthreads();
  for (int i = 0; i < r.count; ++i) {
    float q[8], k[8];
    const f32x4_t* qp = reinterpret_cast<const f32x4_t*>(&qk_lds[i][0][p * 8]);
    const f32x4_t* kp = reinterpret_cast<const f32x4_t*>(&qk_lds[i][1][p * 8]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q[e] = qp[e >> 2][e & 3];
      k[e] = kp[e >> 2][e & 3];
    }
    const float decay = gate_lds[i][0], beta = gate_lds[i][1];
    float yv = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float one = gdn_token(s[c], k, q, v_lds[i][g * NC + c], decay, beta);
      if (p == c) yv = one;
    }
    if (p < NC) yb[i * ystep + g * NC + p] = yv;
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float* to = state + r.write * pool.stride + at + c * kDk;
    *reinterpret_cast<f32x4_t*>(to) = f32x4_t{s[c][0], s[c][1], s[c][2], s[c][3]};
    *reinterpret_cast<f32x4_t*>(to + 4) = f32x4_t{s[c][4], s[c][5], s[c][6], s[c][7]};
  }
}

// ---------------------------------------------------------------------------------------------------------
// The rule in chunks of 32 tokens. With G_i the sum of the log decays up to token i of a chunk and S the state before it,
// the corrections d_i = beta_i (v_i - e^G_i k_i.S - sum_{j<i} e^(G_i - G_j) (k_i.k_j) d_j) are d = T R, where
//   T = (I + L)^-1, L_ij = beta_i e^(G_i - G_j) k_i.k_j (j < i), R_i = beta_i (v_i - e^G_i k_i.S);
//   y_i = e^G_i q_i.S + sum_{j<=i} e^(G_i - G_j) (q_i.k_j) d_j;   S <- e^G_C S + sum_j e^(G_C - G_j) k_j d_j^T.
// So the state is met in matrix products, once a chunk, and a token costs no chain of its own.
//
// A workgroup has WC waves for value columns (16 * NT each, whose states stay in their registers from the first chunk to the
// last) and NP that prepare chunks. A preparing wave takes every NPth chunk, through NP periods between the workgroup's barriers:
// its loads; the products of keys and queries, gates and L; T by substitution; everything into LDS in the matrix cores' operand
// order, for the period after. So one chunk is ready each period, K and Q are read once a workgroup, and no wave waits on memory.
// NP is 4, or 6 where a period's longest piece of preparing would be longer than what one or two waves of 16 columns do in it: then
// the last two are in halves (2039 tokens of 16 heads 131 -> 124 us, 1024 of 64 heads 78 -> 73; with four waves of columns 84 and 84,
// and 8 % slower where workgroups wait for a CU).
//
// Rows of the products are dealt to tokens, and rows of the state to key dims, as 8 (r / 4) + 4 (tile) + r % 4: then what one
// product leaves in a lane (eight consecutive tokens, or dims, of one value column) is the operand that the next one takes.
//
// All of it is held in 32 bits, and so is what a product takes of it: S, R, d, T and the products of q and k are each the sum of
// three bf16 terms, which is all 24 bits of a value down to 2^-110; keys and queries are bf16 as they came, times the power of two
// below their length's inverse. A product of two sums is six products of terms (the others are 2^-22 of it at most). Decays are
// products of the tokens' own, not exponentials of differences, which lose after a strong decay what it has taken.
//
// Fewer bits are faster and do not hold. Two fp16 terms (60 matrix products a chunk and column tile for 96: 97 us where this takes
// 124, 225 for 295) end at 2^-25 of a power of two that a column's values share: where these or the state fall inside a chunk, after
// an outlier or by strong decays, the rows after it lose as many digits (2^-12: 1e-3 off), and setting such powers anew took a state
// that all but vanishes to infinity. Two bf16 terms are 5e-6 off everywhere.
//
// A correction that is not finite (a value, key or gate that is no number; a state that is none) would meet the rows before its
// token as 0 * NaN: such a chunk's columns are taken token by token instead.
//
// Bound by the chains of single waves, of columns and preparing, where heads are few (a prompt of 2039 tokens, 16 heads: 124 us), by
// the issue of two waves a SIMD where they are many (16 prompts of up to 1501 tokens, 32 heads: 295 us, of which a copy's rate would
// take 149).
constexpr int kChunk = 32;

typedef __attribute__((ext_vector_type(2))) uint16_t u16x2_t;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
__device__ __forceinline__ bf16x8_t bf16x8(u32x4_t v) { return __builtin_bit_cast(bf16x8_t, v); }

constexpr int kPitch = 36;  // floats of a row of L and T
struct ChunkScalars {
  float beta[kChunk], in[kChunk], out[kChunk], end[kChunk];  // beta; beta |k| e^G; |q| e^G; |k| e^(G_C - G)
  float decay[kChunk], k[kChunk], q[kChunk];                 // token by token: the factors that make the rows unit vectors
  float total;                                               // e^G_C
  float pad[3];
};
struct ChunkOps {        // 1 KB operands: a lane's 16 bytes after its neighbour's
  u32x4_t k[2][4][64];   // [token tile][dim step]
  u32x4_t q[2][4][64];
  u32x4_t t[3][2][64];   // [term][token tile]
  u32x4_t a[3][2][64];
  ChunkScalars sc;
};
struct ChunkScratch {
  float l[kChunk][kPitch], t[kChunk][kPitch];
  float beta[kChunk], decay[kChunk];
  float inner[kChunk];         // the product of the decays of a token's eight up to it
  float since[kChunk], until[kChunk];  // e^G, e^(G_C - G)
  // of the keys, then the queries: the squares; a power of two near the length's inverse; what that leaves of 1 / sqrt(squares +
  // 1e-6); that
  float sq[2 * kChunk], two[2 * kChunk], rest[2 * kChunk], inv[2 * kChunk];
};
template <int NP>
struct ChunkLds {
  ChunkOps ops[2];
  ChunkScratch scratch[NP];
};

// What one wave's lanes exchange through LDS: written before, read after.
__device__ __forceinline__ void lanes_meet() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The sum over the four quads' values, in every lane.
__device__ __forceinline__ float quads_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The two bf16 halves of a word.
__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Eight values as the sum of three bf16 terms, largest first, exact: eight bits of 24 each. `cut`: a value's first, second and third
// eight bits, by fewer instructions one after the other; else each the nearest. Where both factors of a product are split, one is cut
// and one not, so that what mfma_split leaves out has either sign: 1.4e-7 of the results' norm off (both cut 1.7e-7, none 1.3e-7; 16
// prompts of up to 1501 tokens 298, 296 and 312 us).
struct Split {
  bf16x8_t term[3];
};
template <bool cut>
__device__ __forceinline__ Split split(const float (&v)[8]) {
  u32x4_t w[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      const uint32_t word = cut ? __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u) : two_bf16(a, b);
      w[n][i] = word;
      a -= cut ? high(__float_as_uint(a)) : low(word);
      b -= cut ? high(__float_as_uint(b)) : high(word);
    }
  }
  return {bf16x8(w[0]), bf16x8(w[1]), bf16x8(w[2])};
}

// c + a b, of the six products of terms that hold 24 bits, the smallest first.
__device__ __forceinline__ f32x4_t mfma_split(const bf16x8_t (&a)[3], const bf16x8_t (&b)[3], f32x4_t c) {
  c = mfma16x16x32(a[2], b[0], c);
  c = mfma16x16x32(a[0], b[2], c);
  c = mfma16x16x32(a[1], b[1], c);
  c = mfma16x16x32(a[1], b[0], c);
  c = mfma16x16x32(a[0], b[1], c);
  return mfma16x16x32(a[0], b[0], c);
}

// Whether one of the eight is an infinity or NaN.
__device__ __forceinline__ bool no_numbers(bf16x8_t v) {
  const u32x4_t w = __builtin_bit_cast(u32x4_t, v);
  u16x2_t m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, w[i] & 0x7fff7fffu));
  return m.x >= 0x7f80 || m.y >= 0x7f80;
}

// Lane i - N of the same eight, or 1.
template <int N>
__device__ __forceinline__ float times_before(float v, int lane) {
  const float u = __int_as_float(__builtin_amdgcn_update_dpp(0x3f800000, __float_as_int(v), 0x110 + N, 0xF, 0xF, false));
  return v * ((lane & 7) >= N ? u : 1.f);
}
template <int N>
__device__ __forceinline__ float times_after(float v, int lane) {
  const float u = __int_as_float(__builtin_amdgcn_update_dpp(0x3f800000, __float_as_int(v), 0x100 + N, 0xF, 0xF, false));
  return v * ((lane & 7) + N < 8 ? u : 1.f);
}

// Waits for loads and stores (vmcnt(0)). At the end of a rare path: where it meets the usual one, the compiler would have that one
// wait for all that either may have in flight (7 % of 16 prompts of up to 1501 tokens).
__device__ __forceinline__ void nothing_in_flight() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// v, which the compiler then forms again in every turn of a loop: its sums with other offsets, formed before it, take two
// registers each.
__device__ __forceinline__ uint32_t here(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}
// Eight floats at a multiple of four.
__device__ __forceinline__ void eight_of(const float* of, float (&to)[8]) {
  const f32x4_t a = *reinterpret_cast<const f32x4_t*>(of), b = *reinterpret_cast<const f32x4_t*>(of + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    to[i] = a[i];
    to[4 + i] = b[i];
  }
}

// The waves that prepare chunks: wave `p` the chunks p, p + NP, ... A chunk's gates are asked for a turn ahead.
struct Rows {
  const uint16_t* qkv;  // of the sequence's first token
  uint32_t ldq;
  const uint16_t *b, *a;
  uint32_t ldab;
  int h, hk, H, Hk, count;
};
template <int NP>
__device__ __forceinline__ void prepare_chunks(const Rows& x, ChunkLds<NP>& lds, int p, int chunks, float neg_a, float dtb) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  ChunkScratch& my = lds.scratch[p];
  const int tok[2] = {8 * (r >> 2) + (r & 3), 8 * (r >> 2) + 4 + (r & 3)};  // of this lane's row in each token tile
  uint32_t off[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) off[t] = tok[t] * x.ldq + q * 8;
  const uint32_t goff = min(lane, kChunk - 1) * x.ldab;
  uint16_t na = 0, nb = 0;
  auto load_gates = [&](int c) {
    if (c >= chunks) return;
    const int64_t row = (int64_t)c * kChunk;
    const int live = min(kChunk, x.count - c * kChunk);
    const uint32_t at = live == kChunk ? goff : (uint32_t)min(lane, live - 1) * x.ldab;
    na = (x.a + row * x.ldab + x.h)[at];
    nb = (x.b + row * x.ldab + x.h)[at];
  };
  load_gates(p);
  // Periods: chunk c's last one here is the one before the other waves take it, NP before the first chunk's.
  int left = chunks + NP;
  auto end_period = [&]() {
    lds_barrier();
    --left;
  };
  auto half_period = [&]() {
    if (NP == 6) end_period();
  };
  for (int i = 0; i < p; ++i) end_period();
  for (int c = p; c < chunks; c += NP) {
    const int t0 = c * kChunk, live = min(kChunk, x.count - t0);
    bf16x8_t kf[2][4], qf[2][4];
    Split aq[2];
    {
      {
        const uint16_t* base = x.qkv + (int64_t)t0 * x.ldq + (size_t)x.hk * kDk;
        const uint16_t* kbase = base + (size_t)x.Hk * kDk;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t at = live == kChunk ? off[t] : min(tok[t], live - 1) * x.ldq + q * 8;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            qf[t][s] = *reinterpret_cast<const bf16x8_t*>(base + at + s * 32);
            kf[t][s] = *reinterpret_cast<const bf16x8_t*>(kbase + at + s * 32);
          }
        }
        // A lane per token: its gates, and the products of decays.
        const bool there = lane < live;
        const float decay = there ? expf(neg_a * softplus(bf16_bits_to_f32(na) + dtb)) : 1.f;
        const float beta = there ? 1.0f / (1.0f + expf(-bf16_bits_to_f32(nb))) : 0.f;
        const float inner = times_before<4>(times_before<2>(times_before<1>(decay, lane), lane), lane);
        const float upto = times_after<4>(times_after<2>(times_after<1>(decay, lane), lane), lane);  // from it to its eight's end
        float after = __int_as_float(__builtin_amdgcn_update_dpp(0x3f800000, __float_as_int(upto), 0x101, 0xF, 0xF, false));
        if ((lane & 7) == 7) after = 1.f;
        float block[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) block[i] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(inner), 8 * i + 7));
        const int own = lane >> 3;
        const float first = own == 0 ? 1.f : own == 1 ? block[0] : own == 2 ? block[0] * block[1] : block[0] * block[1] * block[2];
        const float last = own == 0 ? block[1] * block[2] * block[3] : own == 1 ? block[2] * block[3] : own == 2 ? block[3] : 1.f;
        if (lane < kChunk) {
          my.beta[lane] = beta;
          my.decay[lane] = decay;
          my.inner[lane] = inner;
          my.since[lane] = first * inner;
          my.until[lane] = after * last;
        }
      }
      end_period();
      {
        if (live < kChunk) {  // rows past the end
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              const u32x4_t none = {0, 0, 0, 0};
              kf[t][s] = __builtin_bit_cast(bf16x8_t, tok[t] < live ? __builtin_bit_cast(u32x4_t, kf[t][s]) : none);
              qf[t][s] = __builtin_bit_cast(bf16x8_t, tok[t] < live ? __builtin_bit_cast(u32x4_t, qf[t][s]) : none);
            }
        }
        // Rows i = tok[ti] of this lane (its column of the products), columns j = 8q .. 8q + 7.
        f32x4_t kk[2][2], qk[2][2], qq[2];
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
          qq[ti] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < 2; ++t) kk[ti][t] = qk[ti][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int ti = 0; ti < 2; ++ti) {
            qq[ti] = mfma16x16x32(qf[ti][s], qf[ti][s], qq[ti]);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              kk[ti][t] = mfma16x16x32(kf[t][s], kf[ti][s], kk[ti][t]);
              qk[ti][t] = mfma16x16x32(kf[t][s], qf[ti][s], qk[ti][t]);
            }
          }
        if (q == r >> 2) {  // the squares are the products' diagonals
#pragma unroll
          for (int ti = 0; ti < 2; ++ti) {
            const int i = r & 3;
            my.sq[tok[ti]] = i == 0 ? kk[ti][ti][0] : i == 1 ? kk[ti][ti][1] : i == 2 ? kk[ti][ti][2] : kk[ti][ti][3];
            my.sq[kChunk + tok[ti]] = i == 0 ? qq[ti][0] : i == 1 ? qq[ti][1] : i == 2 ? qq[ti][2] : qq[ti][3];
          }
        }
        lanes_meet();
        bool none;  // a row whose squares are past 32 bits' range, which then is one of zeros, as token by token
        {           // a lane per row, keys and queries
          const float ss = my.sq[lane], inv = rsqrtf(ss + 1e-6f);
          none = inv == 0.f;
          const uint32_t bits = __float_as_uint(rsqrtf(fmaxf(ss, 0x1p-126f))) & 0x7f800000u;
          my.two[lane] = __uint_as_float(bits);
          my.rest[lane] = inv * __uint_as_float(0x7f000000u - bits);
          my.inv[lane] = inv;
        }
        lanes_meet();
        if (__any(none)) {  // its products may be infinite
#pragma unroll
          for (int ti = 0; ti < 2; ++ti)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const bool key = my.inv[8 * q + e] == 0.f;
              kk[ti][e >> 2][e & 3] = key || my.inv[tok[ti]] == 0.f ? 0.f : kk[ti][e >> 2][e & 3];
              qk[ti][e >> 2][e & 3] = key || my.inv[kChunk + tok[ti]] == 0.f ? 0.f : qk[ti][e >> 2][e & 3];
            }
        }
        const int mine = r >> 2;  // the eight that holds both rows
        const float between = (q < 1 && mine > 1 ? my.inner[15] : 1.f) * (q < 2 && mine > 2 ? my.inner[23] : 1.f);
        float dj[8], kj[8];
        eight_of(&my.decay[8 * q], dj);
        eight_of(&my.inv[8 * q], kj);
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
          const int i = tok[ti], at = mine == q ? i & 7 : -1;
          const float qn = my.inv[kChunk + i], bk = my.beta[i] * my.inv[i];
          float l[8], a[8];
          float w = mine > q ? my.inner[i] * between : 0.f;  // e^(G_i - G_j), from j = 8q + 7 down
#pragma unroll
          for (int e = 7; e >= 0; --e) {
            w = e == at ? 1.f : w;
            const float wk = w * kj[e];  // (times the product first: two long rows' inverses may leave nothing of each other)
            l[e] = kk[ti][e >> 2][e & 3] * wk * bk;
            a[e] = qk[ti][e >> 2][e & 3] * wk * qn;
            w *= dj[e];
          }
          aq[ti] = split<true>(a);
          // (L's diagonal and what is above it are not read)
          *reinterpret_cast<f32x4_t*>(&my.l[i][8 * q]) = f32x4_t{l[0], l[1], l[2], l[3]};
          *reinterpret_cast<f32x4_t*>(&my.l[i][8 * q + 4]) = f32x4_t{l[4], l[5], l[6], l[7]};
        }
      }
      end_period();
      {
        // T's diagonal blocks of 16 by substitution, a lane per column: row i is e_i less the rows before it times L's. Then the
        // block below: T21 = -T22 (L21 T11), fp32 products whose step k takes rows 4q + k, which the first one leaves in quad q.
        const int half = q & 1;
        float t[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          f32x4_t acc = {i == r ? 1.f : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j0 = 0; j0 < i; j0 += 4) {
            const f32x4_t l = *reinterpret_cast<const f32x4_t*>(&my.l[16 * half + i][16 * half + j0]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j0 + j < i) acc[j] = fmaf(-l[j], t[j0 + j], acc[j]);
          }
          t[i] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
        }
        if (q < 2) {
#pragma unroll
          for (int i = 0; i < 16; ++i) my.t[16 * half + i][16 * half + r] = t[i];
        }
        lanes_meet();
        half_period();
        f32x4_t x = {0.f, 0.f, 0.f, 0.f}, below = x;
        const f32x4_t l21 = *reinterpret_cast<const f32x4_t*>(&my.l[16 + r][4 * q]);
        const f32x4_t t22 = *reinterpret_cast<const f32x4_t*>(&my.t[16 + r][16 + 4 * q]);
#pragma unroll
        for (int k = 0; k < 4; ++k) x = __builtin_amdgcn_mfma_f32_16x16x4f32(l21[k], my.t[4 * q + k][r], x, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) below = __builtin_amdgcn_mfma_f32_16x16x4f32(t22[k], x[k], below, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) my.t[16 + 4 * q + e][r] = -below[e];
      }
      end_period();
      {
        load_gates(c + NP);
        ChunkOps& to = lds.ops[c & 1];
        u32x4_t kh[2][4], qh[2][4];
        Split tt[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float k2 = my.two[tok[t]], q2 = my.two[kChunk + tok[t]];
          auto times = [&](bf16x8_t v, float two) {
            const u32x4_t w = __builtin_bit_cast(u32x4_t, v);
            u32x4_t y;
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = two_bf16(low(w[i]) * two, high(w[i]) * two);
            return y;
          };
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            kh[t][s] = times(kf[t][s], k2);
            qh[t][s] = times(qf[t][s], q2);
          }
          float row[8];
          eight_of(&my.t[tok[t]][8 * q], row);
#pragma unroll
          for (int e = 0; e < 8; ++e) row[e] = tok[t] < 16 && q >= 2 ? 0.f : row[e];
          tt[t] = split<true>(row);
        }
        half_period();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            to.k[t][s][lane] = kh[t][s];
            to.q[t][s][lane] = qh[t][s];
          }
#pragma unroll
          for (int n = 0; n < 3; ++n) {
            to.t[n][t][lane] = __builtin_bit_cast(u32x4_t, tt[t].term[n]);
            to.a[n][t][lane] = __builtin_bit_cast(u32x4_t, aq[t].term[n]);
          }
        }
        if (lane < kChunk) {
          const float beta = my.beta[lane], kr = my.rest[lane], qr = my.rest[kChunk + lane], since = my.since[lane];
          to.sc.beta[lane] = beta;
          to.sc.in[lane] = beta * kr * since;
          to.sc.out[lane] = qr * since;
          to.sc.end[lane] = kr * my.until[lane];
          to.sc.decay[lane] = my.decay[lane];
          to.sc.k[lane] = kr;
          to.sc.q[lane] = qr;
          if (lane == kChunk - 1) to.sc.total = since;
        }
      }
      end_period();
    }
  }
  while (left > 0) end_period();
}

constexpr int kBuffer = 0x00020000;  // a raw buffer's words

template <int WC, int NT, int NP>
__global__ __launch_bounds__(64 * (WC + NP)) void gdn_batch_chunks_kernel(
    Pool pool, const uint16_t* __restrict__ qkv, int64_t ldq, const uint16_t* __restrict__ bcol, const uint16_t* __restrict__ acol,
    int64_t ldab, const float* __restrict__ A_log, const float* __restrict__ dt_bias, float* state, float* __restrict__ y, int T,
    int H, int Hk) {
  constexpr int COLS = 16 * WC * NT, THREADS = 64 * (WC + NP);
  extern __shared__ u32x4_t chunk_lds[];
  ChunkLds<NP>& lds = *reinterpret_cast<ChunkLds<NP>*>(chunk_lds);
  // Heads that follow each other to one die (they take workgroups in turn): value heads of one key head find its rows in that
  // die's cache (8 sequences of 1024 tokens, 32 heads of 16 key heads 5 % less time; a third less read past it).
  const int x = blockIdx.x, h = H % 8 ? x : x % 8 * (H / 8) + x / 8;
  const int b = blockIdx.z, tid = threadIdx.x, wave = wave_id(), lane = tid & 63;
  const int col0 = (int)blockIdx.y * COLS;
  const Run run = run_of(pool, b, T);
  const size_t row0 = (size_t)b * T, ystep = (size_t)H * kDv;
  float* yb = y + (row0 * H + h) * kDv + col0;
  {
    const int first = run.ok ? run.count : 0;
    const float fill = run.ok ? 0.f : __builtin_nanf("");
    for (int i = tid; i < (T - first) * COLS; i += THREADS) yb[(first + i / COLS) * ystep + i % COLS] = fill;
  }
  if (!run.ok || (run.count == 0 && run.read == run.write)) return;
  const int chunks = (run.count + kChunk - 1) / kChunk;
  const uint16_t* rows = qkv + (int64_t)row0 * ldq;
  if (wave >= WC) {
    const Rows seq{rows, (uint32_t)ldq, bcol + (int64_t)row0 * ldab, acol + (int64_t)row0 * ldab, (uint32_t)ldab, h, h / (H / Hk), H, Hk, run.count};
    if (chunks) prepare_chunks(seq, lds, wave - WC, chunks, -expf(A_log[h]), dt_bias[h]);
    return;
  }
  __builtin_amdgcn_s_setprio(1);  // before the preparing waves, which have time to spare: 1 to 2 %
  const int r = lane & 15, q = lane >> 4;
  // of the workgroup's; + nt: a lane's columns are neighbours, and their values (results) one load (store)
  const int col = wave * 16 * NT + NT * r;
  f32x4_t st[NT][4][2];  // dims 32 s + 8 q + 4 half + i of column col + nt
  const size_t at = ((size_t)h * kDv + col0 + col) * kDk + q * 8;
  float* to = state + run.write * pool.stride + at;
  auto get_state = [&](const float* from) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int half = 0; half < 2; ++half) st[nt][s][half] = *reinterpret_cast<const f32x4_t*>(from + nt * kDk + s * 32 + half * 4);
  };
  auto put_state = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          *reinterpret_cast<f32x4_t*>(to + nt * kDk + s * 32 + half * 4) = st[nt][s][half];
  };
  if (run.read >= 0) {
    get_state(state + run.read * pool.stride + at);
  } else {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int half = 0; half < 2; ++half) st[nt][s][half] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const float qscale = rsqrtf((float)kDk);
  // A chunk's values and results as buffers from its first row to the sequence's end, at 32-bit offsets (bytes): loads past it are
  // zero, stores nothing. So no path through a chunk but the rare one below has a branch around either, and the compiler knows at
  // each wait how many are behind it.
  const uint16_t* vrow = rows + (size_t)2 * Hk * kDk + (size_t)h * kDv + col0;
  const uint32_t ld = (uint32_t)ldq * 2, yld = (uint32_t)ystep * 4;
  uint32_t nv[8];  // of the lane's columns, 16 bits each
  auto value = [&](int nt, int e) { return __uint_as_float(nt ? nv[e] & 0xffff0000u : nv[e] << 16); };
  auto load_v = [&](int c) {
    const int left = min(kChunk, run.count - c * kChunk);
    const auto from = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(vrow + (int64_t)c * kChunk * ldq), 0, left * ld, kBuffer);
    uint32_t at = here(8 * q * ld + col * 2);
#pragma unroll
    for (int e = 0; e < 8; ++e, at += ld)
      nv[e] = NT == 1 ? __builtin_amdgcn_raw_buffer_load_b16(from, at, 0, 0) : __builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0);
  };
  if (chunks) {
    load_v(0);
    for (int i = 0; i < NP; ++i) lds_barrier();  // the first chunk's periods
    nothing_in_flight();
  }
  for (int c = 0; c < chunks; ++c) {
    const ChunkOps& ops = lds.ops[c & 1];
    const int t0 = c * kChunk, live = min(kChunk, run.count - t0);
    f32x4_t ks[NT][2], qs[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int t = 0; t < 2; ++t) ks[nt][t] = qs[nt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      Split sp[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const f32x4_t a = st[nt][s][0], d = st[nt][s][1];
        const float eight[8] = {a[0], a[1], a[2], a[3], d[0], d[1], d[2], d[3]};
        sp[nt] = split<true>(eight);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bf16x8_t kf = bf16x8(ops.k[t][s][lane]), qf = bf16x8(ops.q[t][s][lane]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int n = 0; n < 3; ++n) {
            ks[nt][t] = mfma16x16x32(kf, sp[nt].term[n], ks[nt][t]);
            qs[nt][t] = mfma16x16x32(qf, sp[nt].term[n], qs[nt][t]);
          }
      }
    }
    f32x4_t d[NT][2];
    Split dd[NT];
    bool odd = false;
    {
      float beta[8], in[8];
      eight_of(ops.sc.beta + 8 * q, beta);
      eight_of(ops.sc.in + 8 * q, in);
      bf16x8_t tf[2][3];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int n = 0; n < 3; ++n) tf[t][n] = bf16x8(ops.t[n][t][lane]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float right[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) right[e] = fmaf(beta[e], value(nt, e), -in[e] * ks[nt][e >> 2][e & 3]);
        const Split sp = split<false>(right);
#pragma unroll
        for (int t = 0; t < 2; ++t) d[nt][t] = mfma_split(tf[t], sp.term, f32x4_t{0.f, 0.f, 0.f, 0.f});
      }
      if (c + 1 < chunks) load_v(c + 1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float eight[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) eight[e] = d[nt][e >> 2][e & 3];
        dd[nt] = split<false>(eight);
        odd |= no_numbers(dd[nt].term[0]);
      }
    }
    if (!__any(odd)) {
      float out[8], end[8];
      eight_of(ops.sc.out + 8 * q, out);
      eight_of(ops.sc.end + 8 * q, end);
      bf16x8_t af[2][3];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int n = 0; n < 3; ++n) af[t][n] = bf16x8(ops.a[n][t][lane]);
      const auto yr = __builtin_amdgcn_make_buffer_rsrc(yb + (size_t)t0 * ystep, 0, live * yld, kBuffer);
      Split ends[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float decayed[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) decayed[e] = d[nt][e >> 2][e & 3] * end[e];
        ends[nt] = split<true>(decayed);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x4_t& acc = qs[nt][t];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] *= out[4 * t + i];
          acc = mfma_split(af[t], dd[nt].term, acc);
        }
      }
      uint32_t at = here(8 * q * yld + col * 4);
#pragma unroll
      for (int e = 0; e < 8; ++e, at += yld) {
        uint32_t y[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) y[nt] = __float_as_uint(qs[nt][e >> 2][e & 3] * qscale);
        if constexpr (NT == 1) __builtin_amdgcn_raw_buffer_store_b32(y[0], yr, at, 0, 0);
        else __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{y[0], y[1]}, yr, at, 0, 0);
      }
      const float total = ops.sc.total;
      // K turned over, four tokens of a lane's dim at a time: the sixteen lanes of a quad give rows 4q .. 4q + 3 of a tile,
      // four dims each, and take a dim of the four.
      const uint32_t turn = ((4 * q + (r >> 2)) + 16 * (r & 3)) * 16;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          typedef __attribute__((ext_vector_type(4))) short s16x4_t;
          typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
          typedef __attribute__((ext_vector_type(2))) uint32_t two_t;
          two_t part[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const char* from = reinterpret_cast<const char*>(&ops.k[t][s][0]) + turn + 8 * half;
            part[t] = __builtin_bit_cast(two_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)from));
          }
          const bf16x8_t kt = bf16x8(u32x4_t{part[0].x, part[0].y, part[1].x, part[1].y});
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) st[nt][s][half][i] *= total;
#pragma unroll
            for (int n = 2; n >= 0; --n) st[nt][s][half] = mfma16x16x32(kt, ends[nt].term[n], st[nt][s][half]);
          }
        }
    } else {
      // Token by token, on the state in memory, where it ends up anyway: this path is rare, and held in registers it would cost
      // the other one some.
      put_state();
      for (int i = 0; i < live; ++i) {
        const int tile = i >> 2 & 1, row = 4 * (i >> 3) + (i & 3) + 16 * q;
        const float decay = ops.sc.decay[i], kn = ops.sc.k[i], qn = ops.sc.q[i] * qscale, bt = ops.sc.beta[i];
        for (int nt = 0; nt < NT; ++nt) {
          float* mine = to + nt * kDk;
          asm volatile("" ::: "memory");  // the state stays where it is
          float sum = 0.f, yv = 0.f;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const u32x4_t w = ops.k[tile][s][row];
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf((e & 1 ? high(w[e >> 1]) : low(w[e >> 1])) * kn, mine[s * 32 + e], sum);
          }
          const float delta = bt * (bf16_bits_to_f32(vrow[(int64_t)(t0 + i) * ldq + col + nt]) - decay * quads_sum(sum));
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const u32x4_t w = ops.k[tile][s][row], z = ops.q[tile][s][row];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float x = fmaf((e & 1 ? high(w[e >> 1]) : low(w[e >> 1])) * kn, delta, mine[s * 32 + e] * decay);
              mine[s * 32 + e] = x;
              yv = fmaf((e & 1 ? high(z[e >> 1]) : low(z[e >> 1])) * qn, x, yv);
            }
          }
          yv = quads_sum(yv);
          if (q == 0) yb[(size_t)(t0 + i) * ystep + col + nt] = yv;
        }
      }
      asm volatile("" ::: "memory");
      get_state(to);
      nothing_in_flight();
    }
    lds_barrier();
  }
  put_state();
}

template <int WC, int NT, int NP>
int launch_chunks(const Pool& p, const uint16_t* qkv, int64_t ldq, const uint16_t* b, const uint16_t* a, int64_t ldab,
                  const float* A_log, const float* dt_bias, float* state, float* y, int B, int T, int H, int Hk, hipStream_t s) {
  static_assert(sizeof(ChunkLds<NP>) <= 160 * 1024, "a CU's LDS");
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(gdn_batch_chunks_kernel<WC, NT, NP>),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(ChunkLds<NP>));
  if (e != hipSuccess) return skinny_set_error(SKINNY_ELAUNCH, "gdn_batch: %zu bytes of LDS: %s", sizeof(ChunkLds<NP>), hipGetErrorString(e));
  hipLaunchKernelGGL((gdn_batch_chunks_kernel<WC, NT, NP>), dim3(H, kDv / (16 * WC * NT), B), dim3(64 * (WC + NP)),
                     sizeof(ChunkLds<NP>), s, p, qkv, ldq, b, a, ldab, A_log, dt_bias, state, y, T, H, Hk);
  return skinny_check_launch("gdn_batch chunks");
}

int check_pool(const skinny_state_pool* p, int B, int T, int64_t need, Pool& pool, const char* what) {
  SKINNY_CHECK_ARG(p && p->slots, "%s: null pointer", what);
  SKINNY_CHECK_ARG(B >= 1 && B <= 65535 && T >= 1 && T <= 65535, "%s: B=%d sequences of T=%d tokens (1 to 65535 each)",
                   what, B, T);
  SKINNY_CHECK_ARG(p->n_slots >= 1 && p->stride >= need, "%s: n_slots=%d, stride=%lld (a state has %lld elements)", what,
                   p->n_slots, (long long)p->stride, (long long)need);
  SKINNY_CHECK_ARG(skinny_aligned(p->slots, 4) && skinny_aligned(p->slots_out, 4) && skinny_aligned(p->counts, 4),
                   "%s: misaligned slots or counts", what);
  pool = Pool{p->slots, p->slots_out, p->counts, p->n_slots, p->stride};
  return SKINNY_OK;
}

}  // namespace

extern "C" int skinny_gdn_conv_silu_batch(const uint16_t* x, int64_t ldx, int B, int T, int C, int KW,
                                          const skinny_state_pool* pool, uint16_t* conv_state, const uint16_t* weight,
                                          uint16_t* out, int64_t ldo, void* stream) {
  SKINNY_CHECK_ARG(x && conv_state && weight && out, "gdn_conv_batch: null pointer");
  SKINNY_CHECK_ARG(KW == kConvWidth, "gdn_conv_batch: kernel width %d unsupported (only %d)", KW, kConvWidth);
  SKINNY_CHECK_ARG(C >= 1 && C <= (1 << 24) && ldx >= C && ldo >= C, "gdn_conv_batch: bad shape C=%d ldx=%lld ldo=%lld", C,
                   (long long)ldx, (long long)ldo);
  SKINNY_CHECK_ARG(skinny_aligned(x, 2) && skinny_aligned(conv_state, 2) && skinny_aligned(weight, 2) && skinny_aligned(out, 2),
                   "gdn_conv_batch: misaligned buffer");
  Pool p;
  if (const int rc = check_pool(pool, B, T, (int64_t)(KW - 1) * C, p, "gdn_conv_batch")) return rc;
  auto go = [&](auto kernel, int v) {
    const int n = (C + v - 1) / v;
    hipLaunchKernelGGL(kernel, dim3((n + 255) / 256, (T + kTokBlock - 1) / kTokBlock, B), dim3(256), 0, (hipStream_t)stream, p, x,
                       ldx, T, C, conv_state, weight, out, ldo);
  };
  if (C % 2 == 0) go(conv_silu_batch_kernel<2>, 2);
  else go(conv_silu_batch_kernel<1>, 1);
  return skinny_check_launch("gdn_conv_batch");
}

extern "C" int skinny_gdn_recurrence_batch(const uint16_t* qkv, int64_t ldq, const uint16_t* b, const uint16_t* a, int64_t ldab,
                                           const float* A_log, const float* dt_bias, int B, int T,
                                           const skinny_state_pool* pool, float* state, float* y, int H, int Hk, int Dk,
                                           int Dv, void* stream) {
  SKINNY_CHECK_ARG(qkv && b && a && A_log && dt_bias && state && y, "gdn_batch: null pointer");
  SKINNY_CHECK_ARG(Dk == kDk && Dv == kDv, "gdn_batch: head dims %dx%d unsupported (only 128x128)", Dk, Dv);
  SKINNY_CHECK_ARG(H >= 1 && H <= 65535 && Hk >= 1 && H % Hk == 0 && ldq >= (int64_t)2 * Hk * Dk + (int64_t)H * Dv && ldab >= H,
                   "gdn_batch: bad shape H=%d Hk=%d ldq=%lld ldab=%lld", H, Hk, (long long)ldq, (long long)ldab);
  SKINNY_CHECK_ARG(skinny_aligned(qkv, 16) && ldq % 8 == 0, "gdn_batch: qkv rows must be 16-byte aligned");
  SKINNY_CHECK_ARG(ldq < (1 << 25) && ldab < (1 << 25) && (int64_t)H * Dv < (1 << 25),
                   "gdn_batch: rows too far apart");
  SKINNY_CHECK_ARG(skinny_aligned(b, 2) && skinny_aligned(a, 2) && skinny_aligned(A_log, 4) && skinny_aligned(dt_bias, 4) &&
                       skinny_aligned(y, 16),
                   "gdn_batch: misaligned buffer");
  Pool p;
  if (const int rc = check_pool(pool, B, T, (int64_t)H * Dk * Dv, p, "gdn_batch")) return rc;
  SKINNY_CHECK_ARG(skinny_aligned(state, 16) && p.stride % 4 == 0, "gdn_batch: states must be 16-byte aligned");
  if (T > kTokBlock) {
    auto chunks = [&](auto launch) {
      return launch(p, qkv, ldq, b, a, ldab, A_log, dt_bias, state, y, B, T, H, Hk, (hipStream_t)stream);
    };
    // As many workgroups to a head as still find a CU each (their registers leave no room for two): us a call for 16, 32, 64 and
    // 128 columns a workgroup, 1024 tokens of 32 heads: 1 sequence 68 / 71 / 84 / 114, 2 134 / 73 / 84 / 113, 4 265 / 140 / 88 / 113, 8
    // 529 / 279 / 170 / 123.
    const int64_t heads = (int64_t)B * H;
    return heads > 128 ? chunks(launch_chunks<4, 2, 4>) : heads > 64 ? chunks(launch_chunks<4, 1, 4>) : heads > 32 ? chunks(launch_chunks<2, 1, 6>)
                                                                                                             : chunks(launch_chunks<1, 1, 6>);
  }
  auto go = [&](auto kernel, int nc) {
    hipLaunchKernelGGL(kernel, dim3(H, kDv / (kStepGroups * nc), B), dim3(kStepThreads), 0, (hipStream_t)stream, p, qkv, ldq, b, a,
                       ldab, A_log, dt_bias, state, y, T, H, Hk);
  };
  // Columns a lane group, 1 / 2 / 4 / 8, us a call of 32 heads: 16 sequences of 8 tokens 21.9 / 22.1 / 23.9 / 27.6, 64 of 16 109 / 104
  // / 105 / 111; 64 of one token 51.9 / 50.1 / 48.2 / 52.0, 64 of four 57.6 / 51.5 / 51.1 / 56.9.
  if (T <= 4 && (int64_t)B * H >= 1024) go(gdn_batch_steps_kernel<4>, 4);
  else go(gdn_batch_steps_kernel<2>, 2);
  return skinny_check_launch("gdn_batch");
}
