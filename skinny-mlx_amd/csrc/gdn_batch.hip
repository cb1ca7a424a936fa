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
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));

// ---------------------------------------------------------------------------------------------------------
// The conv: a thread per V channels and block of kTokBlock tokens. A token's taps are input rows, or for the first three
// the state's, so the blocks need nothing of each other; the first one reads the state and writes the one after the call.
// Taps oldest first and the exact exponential, as gdn.hip's conv: the same bits. Bound by memory for prompts.
constexpr int kConvWidth = 4;

template <int V>
struct Chans {
  uint32_t w[(V + 1) / 2];
  __device__ __forceinline__ void load(const uint16_t* p) {
    if constexpr (V == 8) {
      const u32x4_t x = *reinterpret_cast<const u32x4_any_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = x[i];
    } else {
      w[0] = *p;
    }
  }
  __device__ __forceinline__ void store(uint16_t* p) const {
    if constexpr (V == 8) *reinterpret_cast<u32x4_any_t*>(p) = u32x4_t{w[0], w[1], w[2], w[3]};
    else *p = (uint16_t)w[0];
  }
  __device__ __forceinline__ void fill(uint32_t half) {
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) w[i] = half * 0x10001u;
  }
  __device__ __forceinline__ float value(int e) const { return bf16_bits_to_f32(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu); }
};

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
  uint16_t taps[V * kConvWidth];
#pragma unroll
  for (int i = 0; i < V * kConvWidth; ++i) taps[i] = weight[(size_t)c * kConvWidth + i];
#pragma unroll
  for (int i = 0; i < kTokBlock; ++i)
    if (i < live) line[H + i].load(x + (int64_t)(t0 + i) * ldx);
#pragma unroll
  for (int i = 0; i < kTokBlock; ++i) {
    if (i >= rows) break;
    Chans<V> y;
    if (i < live) {
      uint16_t half[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float acc = 0.f;
#pragma unroll
        for (int j = 0; j < kConvWidth; ++j) acc = fmaf(bf16_bits_to_f32(taps[e * kConvWidth + j]), line[i + j].value(e), acc);
        half[e] = f32_to_bf16_bits(acc / (1.0f + expf(-acc)));
      }
      if constexpr (V == 1) y.w[0] = half[0];
      else
#pragma unroll
        for (int e = 0; e < V / 2; ++e) y.w[e] = half[2 * e] | (uint32_t)half[2 * e + 1] << 16;
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
    else v = at == 0 ? line[0] : at == 1 ? line[1] : line[2];
    v.store(to + (int64_t)j * C);
  }
}

// ---------------------------------------------------------------------------------------------------------
// The rule token by token: 16 lanes hold a value column (8 key dims each), a group of lanes NC columns, so a workgroup
// 16 * NC of a head's 128. All of the state's loads are issued at once. The token's update is gdn.hip's, its sums in the
// same order: y and the state have the bits of skinny_gdn_recurrence on each sequence alone.
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
  for (int t0 = 0; t0 < r.count; t0 += kTokBlock) {
    const int mb = min(kTokBlock, r.count - t0);
    if (t0 > 0) __syncthreads();
    if (g < mb) {  // a lane group per token: its q and k, normalised
      const uint16_t* row = qkv + (int64_t)(row0 + t0 + g) * ldq + (size_t)hk * kDk + p * 8;
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
        const float x = bf16_bits_to_f32((p ? bcol : acol)[(int64_t)(row0 + t0 + g) * ldab + h]);
        gate_lds[g][p] = p ? 1.0f / (1.0f + expf(-x)) : expf(neg_a * softplus(x + dtb));
      }
    }
    for (int i = tid; i < mb * COLS; i += kStepThreads)
      v_lds[i / COLS][i % COLS] =
          bf16_bits_to_f32(qkv[(int64_t)(row0 + t0 + i / COLS) * ldq + (size_t)2 * Hk * kDk + (size_t)h * kDv + col0 + i % COLS]);
    __syncthreads();
    for (int i = 0; i < mb; ++i) {
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
      if (p < NC) yb[(t0 + i) * ystep + g * NC + p] = yv;
    }
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
// last) and four that prepare chunks. A preparing wave takes every fourth chunk, through four periods between the workgroup's
// barriers: its loads; the products of keys and queries, gates and L; T by substitution; everything into LDS in the matrix
// cores' operand order, for the period after. So one chunk is ready each period, K and Q are read once a workgroup, and no
// wave waits on memory.
//
// Rows of the products are dealt to tokens, and rows of the state to key dims, as 8 (r / 4) + 4 (tile) + r % 4: then what one
// product leaves in a lane (eight consecutive tokens, or dims, of one value column) is the operand that the next one takes.
//
// All of it is held in 32 bits. K and Q go in as they are, in bf16, their norms applied to the products in 32 bits; S, R, d, T
// and the products of q and k are taken as the sum of two bf16 terms (2^-16 of each), so a term's 2^-8 is in no result. G is
// summed in 64 bits: e^(G_i - G_j) of two tokens after a strong decay would otherwise lose what the decay has taken.
//
// A correction that is not finite (a value, key or gate that is no number; a state that is none) would meet the rows before its
// token as 0 * NaN: such a chunk's columns are taken token by token instead.
constexpr int kChunk = 32, kProducers = 4;
constexpr float kNoDecay = -110.f;  // e^-110 is zero in 32 bits; sums of what is below would only lose digits

constexpr int kPitch = 36;  // floats of a row of L and T
struct ChunkScalars {
  float beta[kChunk], in[kChunk], out[kChunk], end[kChunk];  // beta; beta |k| e^G; |q| e^G; |k| e^(G_C - G)
  float decay[kChunk], kn[kChunk], qn[kChunk];               // token by token
  float total;                                               // e^G_C
  float pad[3];
};
struct ChunkOps {          // 1 KB operands: a lane's 16 bytes after its neighbour's
  u32x4_t k[2][4][64];     // [token tile][dim step]
  u32x4_t q[2][4][64];
  u32x4_t kt[4][2][64];    // [dim step][half]: rows are key dims
  u32x4_t t[2][2][64];     // [term][token tile]
  u32x4_t a[2][2][64];
  ChunkScalars sc;
};
struct ChunkScratch {
  float l[kChunk][kPitch], t[kChunk][kPitch];
  double g[kChunk];  // log2 of the decays' product
  float beta[kChunk], decay[kChunk], kn[kChunk], qn[kChunk];
};
struct ChunkLds {
  ChunkOps ops[2];
  ChunkScratch scratch[kProducers];
};

// What one wave's lanes exchange through LDS: written before, read after.
__device__ __forceinline__ void lanes_meet() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ float quads_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Eight values as the sum of two bf16 terms.
struct Split {
  bf16x8_t hi, lo;
};
__device__ __forceinline__ Split split(const float (&v)[8]) {
  typedef __attribute__((ext_vector_type(2))) float f32x2_t;
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
  u32x4_t hi, lo;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    hi[w] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{v[2 * w], v[2 * w + 1]}, bf16x2_t));
    const f32x2_t rest = {v[2 * w] - __uint_as_float(hi[w] << 16), v[2 * w + 1] - __uint_as_float(hi[w] & 0xffff0000u)};
    lo[w] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, bf16x2_t));
  }
  return {__builtin_bit_cast(bf16x8_t, hi), __builtin_bit_cast(bf16x8_t, lo)};
}

// The four waves that prepare chunks: wave `p` the chunks p, p + 4, ...
struct Rows {
  const uint16_t* qkv;  // of the sequence's first token
  int64_t ldq;
  const uint16_t *b, *a;
  int64_t ldab;
  int h, hk, H, Hk, count;
};
__device__ __forceinline__ void prepare_chunks(const Rows& x, ChunkLds& lds, int p, int chunks, float neg_a, float dtb) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  ChunkScratch& my = lds.scratch[p];
  const int tok[2] = {8 * (r >> 2) + (r & 3), 8 * (r >> 2) + 4 + (r & 3)};  // of this lane's row in each token tile
  bf16x8_t kf[2][4], qf[2][4];
  Split aq[2];
  uint16_t na = 0, nb = 0;
  for (int n = chunks ? -kProducers : 0; n < chunks; ++n) {
    const int ahead = (p - n - 1) & 3, c = n + 1 + ahead;  // the chunk, `ahead` periods before its last phase
    if (c < chunks && c >= 0) {
      const int t0 = c * kChunk, live = min(kChunk, x.count - t0);
      if (ahead == 3) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint16_t* row = x.qkv + (int64_t)(t0 + min(tok[t], live - 1)) * x.ldq + (size_t)x.hk * kDk + q * 8;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            qf[t][s] = *reinterpret_cast<const bf16x8_t*>(row + s * 32);
            kf[t][s] = *reinterpret_cast<const bf16x8_t*>(row + (size_t)x.Hk * kDk + s * 32);
          }
        }
        const int64_t g = (int64_t)(t0 + min(lane, live - 1)) * x.ldab + x.h;
        na = x.a[g];
        nb = x.b[g];
      } else if (ahead == 2) {
        float kn[2], qn[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float kk = 0.f, qq = 0.f;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            u32x4_t kw = __builtin_bit_cast(u32x4_t, kf[t][s]), qw = __builtin_bit_cast(u32x4_t, qf[t][s]);
            if (tok[t] >= live) kw = qw = u32x4_t{0, 0, 0, 0};  // past the end
            kf[t][s] = __builtin_bit_cast(bf16x8_t, kw);
            qf[t][s] = __builtin_bit_cast(bf16x8_t, qw);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const float k0 = __uint_as_float(kw[w] << 16), k1 = __uint_as_float(kw[w] & 0xffff0000u);
              const float q0 = __uint_as_float(qw[w] << 16), q1 = __uint_as_float(qw[w] & 0xffff0000u);
              kk = fmaf(k0, k0, kk);
              kk = fmaf(k1, k1, kk);
              qq = fmaf(q0, q0, qq);
              qq = fmaf(q1, q1, qq);
            }
          }
          kn[t] = rsqrtf(quads_sum(kk) + 1e-6f);
          qn[t] = rsqrtf(quads_sum(qq) + 1e-6f) * rsqrtf((float)kDk);
          if (q == 0) {
            my.kn[tok[t]] = kn[t];
            my.qn[tok[t]] = qn[t];
          }
        }
        {  // a lane per token
          float g = neg_a * softplus(bf16_bits_to_f32(na) + dtb), beta = 1.0f / (1.0f + expf(-bf16_bits_to_f32(nb)));
          const bool there = lane < live;
          const float decay = there ? expf(g) : 1.f;
          g = there ? (g < kNoDecay ? kNoDecay : g) : 0.f;
          double sum = (double)g * 1.4426950408889634;
#pragma unroll
          for (int step = 1; step < kChunk; step *= 2) {
            const double before = __shfl_up(sum, step, 64);
            if (lane >= step) sum += before;
          }
          if (lane < kChunk) {
            my.g[lane] = sum;
            my.beta[lane] = there ? beta : 0.f;
            my.decay[lane] = decay;
          }
        }
        lanes_meet();
        double gj[8];
        float knj[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          gj[e] = my.g[8 * q + e];
          knj[e] = my.kn[8 * q + e];
        }
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {  // rows i = tok[ti], columns j = 8q .. 8q + 7
          f32x4_t kk[2], qk[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            kk[t] = qk[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              kk[t] = mfma16x16x32(kf[t][s], kf[ti][s], kk[t]);
              qk[t] = mfma16x16x32(kf[t][s], qf[ti][s], qk[t]);
            }
          }
          const double gi = my.g[tok[ti]];
          const float bk = my.beta[tok[ti]] * kn[ti];
          float l[8], a[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int j = 8 * q + e;
            const float w = knj[e] * __builtin_amdgcn_exp2f((float)(gi - gj[e]));
            l[e] = j < tok[ti] ? kk[e >> 2][e & 3] * w * bk : 0.f;
            a[e] = j <= tok[ti] ? qk[e >> 2][e & 3] * w * qn[ti] : 0.f;
          }
          aq[ti] = split(a);
          *reinterpret_cast<f32x4_t*>(&my.l[tok[ti]][8 * q]) = f32x4_t{l[0], l[1], l[2], l[3]};
          *reinterpret_cast<f32x4_t*>(&my.l[tok[ti]][8 * q + 4]) = f32x4_t{l[4], l[5], l[6], l[7]};
        }
      } else if (ahead == 1) {
        // T's diagonal blocks of 16 by substitution, a lane per column: row i is e_i less the rows before it times L's. Then the
        // block below: T21 = -T22 (L21 T11), four rows a quad.
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
        auto four_rows = [&](const float (*m)[kPitch], int row, int mcol, int vcol, float (&sum)[4]) {
          float v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = my.t[j][vcol];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j0 = 0; j0 < 16; j0 += 4) {
              const f32x4_t w = *reinterpret_cast<const f32x4_t*>(&m[row + e][mcol + j0]);
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[j] = fmaf(w[j], v[j0 + j], acc[j]);
            }
            sum[e] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
          }
        };
        float four[4];
        four_rows(my.l, 16 + 4 * q, 0, r, four);
#pragma unroll
        for (int e = 0; e < 4; ++e) my.t[4 * q + e][16 + r] = four[e];  // T's upper block, which is zero and not stored
        lanes_meet();
        four_rows(my.t, 16 + 4 * q, 16, 16 + r, four);
#pragma unroll
        for (int e = 0; e < 4; ++e) my.t[16 + 4 * q + e][r] = -four[e];
      } else {
        ChunkOps& to = lds.ops[c & 1];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            to.k[t][s][lane] = __builtin_bit_cast(u32x4_t, kf[t][s]);
            to.q[t][s][lane] = __builtin_bit_cast(u32x4_t, qf[t][s]);
          }
          float row[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) row[e] = tok[t] < 16 && q >= 2 ? 0.f : my.t[tok[t]][8 * q + e];
          const Split two = split(row);
          to.t[0][t][lane] = __builtin_bit_cast(u32x4_t, two.hi);
          to.t[1][t][lane] = __builtin_bit_cast(u32x4_t, two.lo);
          to.a[0][t][lane] = __builtin_bit_cast(u32x4_t, aq[t].hi);
          to.a[1][t][lane] = __builtin_bit_cast(u32x4_t, aq[t].lo);
        }
        if (lane < kChunk) {
          const float since = __builtin_amdgcn_exp2f((float)my.g[lane]);
          const float until = __builtin_amdgcn_exp2f((float)(my.g[kChunk - 1] - my.g[lane]));
          const float beta = my.beta[lane], kn = my.kn[lane], qn = my.qn[lane];
          to.sc.beta[lane] = beta;
          to.sc.in[lane] = beta * kn * since;
          to.sc.out[lane] = qn * since;
          to.sc.end[lane] = kn * until;
          to.sc.decay[lane] = my.decay[lane];
          to.sc.kn[lane] = kn;
          to.sc.qn[lane] = qn;
          if (lane == kChunk - 1) to.sc.total = since;
        }
        lanes_meet();
        // K turned over: row r of (s, half) is dim 32 s + 8 (r / 4) + 4 half + r % 4, its operand tokens 8q .. 8q + 7.
        const uint16_t* k = reinterpret_cast<const uint16_t*>(&to.k[0][0][0]);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            u32x4_t v;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t two[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int e = 2 * w + i;
                two[i] = k[(((e >> 2) * 4 + s) * 64 + 4 * q + (e & 3) + 16 * (r >> 2)) * 8 + 4 * half + (r & 3)];
              }
              v[w] = two[0] | two[1] << 16;
            }
            to.kt[s][half][lane] = v;
          }
      }
    }
    lds_barrier();
  }
}

template <int WC, int NT>
__global__ __launch_bounds__(64 * (WC + kProducers)) void gdn_batch_chunks_kernel(
    Pool pool, const uint16_t* __restrict__ qkv, int64_t ldq, const uint16_t* __restrict__ bcol, const uint16_t* __restrict__ acol,
    int64_t ldab, const float* __restrict__ A_log, const float* __restrict__ dt_bias, float* state, float* __restrict__ y, int T,
    int H, int Hk) {
  constexpr int COLS = 16 * WC * NT, THREADS = 64 * (WC + kProducers);
  extern __shared__ u32x4_t chunk_lds[];
  ChunkLds& lds = *reinterpret_cast<ChunkLds*>(chunk_lds);
  const int h = blockIdx.x, b = blockIdx.z, tid = threadIdx.x, wave = wave_id(), lane = tid & 63;
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
    const Rows x{rows, ldq, bcol + (int64_t)row0 * ldab, acol + (int64_t)row0 * ldab, ldab, h, h / (H / Hk), H, Hk, run.count};
    prepare_chunks(x, lds, wave - WC, chunks, -expf(A_log[h]), dt_bias[h]);
    return;
  }
  const int r = lane & 15, q = lane >> 4;
  const int col = wave * 16 * NT + r;  // of the workgroup's; + 16 nt
  // dims 32 s + 8 q + 4 half + i of column col + 16 nt
  f32x4_t st[NT][4][2];
  const size_t at = ((size_t)h * kDv + col0 + col) * kDk + q * 8;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        st[nt][s][half] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if (run.read >= 0)
          st[nt][s][half] = *reinterpret_cast<const f32x4_t*>(state + run.read * pool.stride + at + (size_t)nt * 16 * kDk + s * 32 + half * 4);
      }
  const uint16_t* vrow = rows + (size_t)2 * Hk * kDk + (size_t)h * kDv + col0 + col;
  uint16_t nv[NT][8];
  auto load_v = [&](int c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t* from = vrow + (int64_t)min(c * kChunk + 8 * q + e, run.count - 1) * ldq;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) nv[nt][e] = from[nt * 16];
    }
  };
  if (chunks) {
    load_v(0);
    for (int i = 0; i < kProducers; ++i) lds_barrier();  // the first chunk's four periods
  }
  for (int c = 0; c < chunks; ++c) {
    const ChunkOps& ops = lds.ops[c & 1];
    const int t0 = c * kChunk, live = min(kChunk, run.count - t0);
    float v[NT][8];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[nt][e] = 8 * q + e < live ? bf16_bits_to_f32(nv[nt][e]) : 0.f;
    if (c + 1 < chunks) load_v(c + 1);
    f32x4_t ks[NT][2], qs[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int t = 0; t < 2; ++t) ks[nt][t] = qs[nt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      Split two[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const f32x4_t a = st[nt][s][0], d = st[nt][s][1];
        const float eight[8] = {a[0], a[1], a[2], a[3], d[0], d[1], d[2], d[3]};
        two[nt] = split(eight);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bf16x8_t kf = __builtin_bit_cast(bf16x8_t, ops.k[t][s][lane]), qf = __builtin_bit_cast(bf16x8_t, ops.q[t][s][lane]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          ks[nt][t] = mfma16x16x32(kf, two[nt].hi, ks[nt][t]);
          qs[nt][t] = mfma16x16x32(qf, two[nt].hi, qs[nt][t]);
          ks[nt][t] = mfma16x16x32(kf, two[nt].lo, ks[nt][t]);
          qs[nt][t] = mfma16x16x32(qf, two[nt].lo, qs[nt][t]);
        }
      }
    }
    auto scalars = [&](const float* of, float (&to)[8]) {
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(of + 8 * q), d = *reinterpret_cast<const f32x4_t*>(of + 8 * q + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        to[i] = a[i];
        to[4 + i] = d[i];
      }
    };
    float beta[8], in[8];
    scalars(ops.sc.beta, beta);
    scalars(ops.sc.in, in);
    f32x4_t d[NT][2];
    bool odd = false;
    {
      bf16x8_t tf[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t) tf[i][t] = __builtin_bit_cast(bf16x8_t, ops.t[i][t][lane]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float right[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) right[e] = fmaf(beta[e], v[nt][e], -in[e] * ks[nt][e >> 2][e & 3]);
        const Split two = split(right);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          d[nt][t] = mfma16x16x32(tf[0][t], two.lo, f32x4_t{0.f, 0.f, 0.f, 0.f});
          d[nt][t] = mfma16x16x32(tf[1][t], two.hi, d[nt][t]);
          d[nt][t] = mfma16x16x32(tf[0][t], two.hi, d[nt][t]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) odd |= !(fabsf(d[nt][e >> 2][e & 3]) < INFINITY);
      }
    }
    if (!__any(odd)) {
      float out[8], end[8];
      scalars(ops.sc.out, out);
      scalars(ops.sc.end, end);
      bf16x8_t af[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t) af[i][t] = __builtin_bit_cast(bf16x8_t, ops.a[i][t][lane]);
      Split ends[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float eight[8], decayed[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          eight[e] = d[nt][e >> 2][e & 3];
          decayed[e] = eight[e] * end[e];
        }
        const Split two = split(eight);
        ends[nt] = split(decayed);
        float* yr = yb + (size_t)(t0 + 8 * q) * ystep + col + 16 * nt;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x4_t acc;
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] = qs[nt][t][i] * out[4 * t + i];
          acc = mfma16x16x32(af[0][t], two.lo, acc);
          acc = mfma16x16x32(af[1][t], two.hi, acc);
          acc = mfma16x16x32(af[0][t], two.hi, acc);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (8 * q + 4 * t + i < live) yr[(4 * t + i) * ystep] = acc[i];
        }
      }
      const float total = ops.sc.total;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const bf16x8_t kt = __builtin_bit_cast(bf16x8_t, ops.kt[s][half][lane]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) st[nt][s][half][i] *= total;
            st[nt][s][half] = mfma16x16x32(kt, ends[nt].lo, st[nt][s][half]);
            st[nt][s][half] = mfma16x16x32(kt, ends[nt].hi, st[nt][s][half]);
          }
        }
    } else {
      for (int i = 0; i < live; ++i) {  // token by token
        const int tile = i >> 2 & 1, row = 4 * (i >> 3) + (i & 3) + 16 * q;
        const float decay = ops.sc.decay[i], kn = ops.sc.kn[i], qn = ops.sc.qn[i], bt = ops.sc.beta[i];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float sum = 0.f;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const u32x4_t w = ops.k[tile][s][row];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              sum = fmaf(bf16_bits_to_f32(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu) * kn, st[nt][s][e >> 2][e & 3], sum);
          }
          const float delta = bt * (bf16_bits_to_f32(vrow[(int64_t)(t0 + i) * ldq + nt * 16]) - decay * quads_sum(sum));
          float yv = 0.f;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const u32x4_t w = ops.k[tile][s][row], z = ops.q[tile][s][row];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float x = fmaf(bf16_bits_to_f32(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu) * kn, delta,
                                   st[nt][s][e >> 2][e & 3] * decay);
              st[nt][s][e >> 2][e & 3] = x;
              yv = fmaf(bf16_bits_to_f32(e & 1 ? z[e >> 1] >> 16 : z[e >> 1] & 0xffffu) * qn, x, yv);
            }
          }
          yv = quads_sum(yv);
          if (q == 0) yb[(size_t)(t0 + i) * ystep + col + 16 * nt] = yv;
        }
      }
    }
    lds_barrier();
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        *reinterpret_cast<f32x4_t*>(state + run.write * pool.stride + at + (size_t)nt * 16 * kDk + s * 32 + half * 4) = st[nt][s][half];
}

template <int WC, int NT>
int launch_chunks(const Pool& p, const uint16_t* qkv, int64_t ldq, const uint16_t* b, const uint16_t* a, int64_t ldab,
                  const float* A_log, const float* dt_bias, float* state, float* y, int B, int T, int H, int Hk, hipStream_t s) {
  static_assert(sizeof(ChunkLds) <= 160 * 1024, "a CU's LDS");
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(gdn_batch_chunks_kernel<WC, NT>),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(ChunkLds));
  if (e != hipSuccess) return skinny_set_error(SKINNY_ELAUNCH, "gdn_batch: %zu bytes of LDS: %s", sizeof(ChunkLds), hipGetErrorString(e));
  hipLaunchKernelGGL((gdn_batch_chunks_kernel<WC, NT>), dim3(H, kDv / (16 * WC * NT), B), dim3(64 * (WC + kProducers)),
                     sizeof(ChunkLds), s, p, qkv, ldq, b, a, ldab, A_log, dt_bias, state, y, T, H, Hk);
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
  if (C % 8 == 0) go(conv_silu_batch_kernel<8>, 8);
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
    const int64_t heads = (int64_t)B * H;
    return heads >= 256 ? chunks(launch_chunks<4, 2>) : heads >= 128 ? chunks(launch_chunks<4, 1>) : chunks(launch_chunks<2, 1>);
  }
  auto go = [&](auto kernel, int nc) {
    hipLaunchKernelGGL(kernel, dim3(H, kDv / (kStepGroups * nc), B), dim3(kStepThreads), 0, (hipStream_t)stream, p, qkv, ldq, b, a,
                       ldab, A_log, dt_bias, state, y, T, H, Hk);
  };
  if ((int64_t)B * H >= 512) go(gdn_batch_steps_kernel<8>, 8);
  else go(gdn_batch_steps_kernel<1>, 1);
  return skinny_check_launch("gdn_batch");
}
