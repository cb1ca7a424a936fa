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
  auto go = [&](auto kernel, int nc) {
    hipLaunchKernelGGL(kernel, dim3(H, kDv / (kStepGroups * nc), B), dim3(kStepThreads), 0, (hipStream_t)stream, p, qkv, ldq, b, a,
                       ldab, A_log, dt_bias, state, y, T, H, Hk);
  };
  if ((int64_t)B * H >= 512) go(gdn_batch_steps_kernel<8>, 8);
  else go(gdn_batch_steps_kernel<1>, 1);
  return skinny_check_launch("gdn_batch");
}
