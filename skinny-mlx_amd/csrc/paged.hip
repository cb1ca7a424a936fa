// A key-value cache in pages shared by several sequences, and the attention of each sequence's new tokens
// over it: the batched counterpart of the contiguous caches of attn.hip and attn_general.hip.
//
// No reference counterpart: the reference decodes one sequence (skinny_mlx/spec.py:98-156). Arithmetic of a
// layer as at spec.py:24-29 (per-head q/k RMSNorm, rotate-half RoPE over the first R dims, causal GQA
// attention, optionally output * sigmoid(gate)).
//
// Pages: K [page][Hkv][P][D] and V transposed [page][Hkv][D][P], P a power of two from 16 to 256, so a
// head's part of a page is one contiguous run of P * D values in both, and eight consecutive keys of one
// dim are one 16-byte piece, as the matrix cores take them. Sequence b holds lengths[b] tokens before the
// call and brings counts[b] of at most T new ones, at positions lengths[b] + t; position p lives in slot
// p % P of page pages[b][p / P].
#include "common.h"

namespace {

constexpr float kPLog2e = 1.4426950408889634f;
constexpr int kPWaves = 4;      // waves of an attention workgroup: one run of atom keys each
constexpr int kPMaxRows = 64;   // query rows per kv head: T x (Hq / Hkv)
constexpr int kPMergeWaves = 4;

// Keys that one wave takes at once: 32 KB of K and V at 128 and 256 dims, held in registers.
__host__ __device__ constexpr int paged_atom(int D) { return D == 256 ? 32 : 64; }
__host__ __device__ constexpr int paged_block(int D) { return paged_atom(D) * kPWaves; }

struct Pages {
  const int32_t* lengths;
  const int32_t* counts;  // null: T each
  const int32_t* table;   // [B][>= max_pages], row stride ld
  uint16_t* k;
  uint16_t* vt;
  int64_t k_stride, vt_stride;  // elements from page to page
  int ld, n_pages, log2p;
};

// A sequence's cached length and new tokens. `ok` is false where they cannot be: a negative length, a count
// outside [0, T], or more tokens than `room` slots.
struct Sequence {
  int len, count;
  bool ok;
};
__device__ __forceinline__ Sequence sequence_of(const Pages& pg, int b, int T, int room) {
  const int len = pg.lengths[b], count = pg.counts ? pg.counts[b] : T;
  return {len, count, len >= 0 && count >= 0 && count <= T && count <= room && len <= room - count};
}

constexpr uint16_t kNanBits = 0x7fc0;

// ---------------------------------------------------------------------------------------------------------
// New rows into the cache.

// One wave per (head, token, sequence): heads [0, Hq) are queries, then Hkv keys, then Hkv values. Lane l holds dims
// l + 64e. fp32 from the row to the result, rounded once.
template <int D>
__global__ __launch_bounds__(64) void paged_store_kernel(Pages pg, const uint16_t* __restrict__ qkv, int ldq, int T,
                                                         int Hq, int Hkv, int qs, int koff, int voff,
                                                         const uint16_t* __restrict__ qn, const uint16_t* __restrict__ kn,
                                                         float eps, int R, const float* __restrict__ rope, int room,
                                                         uint16_t* __restrict__ q_out) {
  constexpr int E = D / 64;
  __shared__ float row[D];
  const int head = blockIdx.x, t = blockIdx.y, b = blockIdx.z, lane = threadIdx.x;
  const Sequence sq = sequence_of(pg, b, T, room);
  const size_t r = (size_t)b * T + t;
  uint16_t* qd = q_out + (r * Hq + head) * D;
  const bool live = sq.ok && t < sq.count;
  const int pos = live ? sq.len + t : 0;
  const int P = 1 << pg.log2p;
  int page = -1;
  if (live) page = pg.table[(size_t)b * pg.ld + (pos >> pg.log2p)];
  const bool placed = (unsigned)page < (unsigned)pg.n_pages;
  if (!live || !placed) {
    if (head < Hq) {
      const uint16_t fill = sq.ok && t >= sq.count ? 0 : kNanBits;
#pragma unroll
      for (int e = 0; e < E; ++e) qd[lane + 64 * e] = fill;
    }
    return;
  }
  const uint16_t* src = qkv + r * ldq;
  if (head < Hq) src += (size_t)head * qs;
  else if (head < Hq + Hkv) src += koff + (head - Hq) * D;
  else src += voff + (head - Hq - Hkv) * D;
  const int slot = pos & (P - 1);
  if (head >= Hq + Hkv) {
    uint16_t* vd = pg.vt + (int64_t)page * pg.vt_stride + (size_t)(head - Hq - Hkv) * D * P + slot;
#pragma unroll
    for (int e = 0; e < E; ++e) vd[(size_t)(lane + 64 * e) * P] = src[lane + 64 * e];
    return;
  }
  float x[E];
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[e] = bf16_bits_to_f32(src[lane + 64 * e]);
    ss = fmaf(x[e], x[e], ss);
  }
  const uint16_t* nw = head < Hq ? qn : kn;
  if (nw) {
    const float inv = rsqrtf(wave_sum(ss) / (float)D + eps);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] *= inv * bf16_bits_to_f32(nw[lane + 64 * e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) row[lane + 64 * e] = x[e];
  __syncthreads();
  const int half = R >> 1;
  uint16_t* dst = head < Hq ? qd : pg.k + (int64_t)page * pg.k_stride + ((size_t)(head - Hq) * P + slot) * D;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 64 * e;
    float y = x[e];
    if (d < R) {
      const int i = d < half ? d : d - half;
      const float2 cs = reinterpret_cast<const float2*>(rope)[(size_t)pos * half + i];
      const float a = row[i], c = row[i + half];
      y = d < half ? a * cs.x - c * cs.y : c * cs.x + a * cs.y;
    }
    dst[d] = f32_to_bf16_bits(y);
  }
}

// ---------------------------------------------------------------------------------------------------------
// Attention. A block of paged_block(D) keys of one sequence and kv head is one workgroup's: each wave takes an
// atom of paged_atom(D) keys straight from memory into matrix-core operands, S^T = K Q^T, an exact softmax of the
// atom, O^T = V^T P^T, and the four atoms are folded in order. Blocks are joined in order by the merge. Atoms and
// blocks are cut at fixed positions of the sequence, and a row that does not see an atom adds nothing to it, so a
// row's bits depend on its own sequence and position alone: not on the batch, on T, or on where the pages lie.

// The first n (0 to 8) of eight consecutive keys' values, the others zero.
__device__ __forceinline__ u32x4_t first_keys(u32x4_t v, int n) {
#pragma unroll
  for (int w = 0; w < 4; ++w)
    v[w] &= (2 * w < n ? 0xffffu : 0u) | (2 * w + 1 < n ? 0xffff0000u : 0u);
  return v;
}

struct Out {
  uint16_t* out;
  const uint16_t* gate;  // null: none
  int64_t ldg;           // elements from row to row
  int gs;                // and from head to head
};

// One output value o / l, gated, rounded.
__device__ __forceinline__ uint16_t finished(float o, float l, const uint16_t* gate, int d) {
  o /= l;
  if (gate) o /= 1.f + __builtin_amdgcn_exp2f(bf16_bits_to_f32(gate[d]) * -kPLog2e);
  return f32_to_bf16_bits(o);
}

template <int D>
__global__ __launch_bounds__(64 * kPWaves, 2) void paged_block_kernel(Pages pg, const uint16_t* __restrict__ q, int T,
                                                                      int Hq, int Hkv, int room, float scale, int nblk,
                                                                      float* __restrict__ part_o,
                                                                      float* __restrict__ part_ml, Out o) {
  constexpr int ATOM = paged_atom(D), BLK = paged_block(D);
  constexpr int KS = D / 32, DT = D / 16, KT = ATOM / 16, PS = ATOM / 32, GR = ATOM / 16;
  constexpr int OP = D + 4;  // LDS pitch of an output row
  __shared__ __attribute__((aligned(16))) float o_lds[kPWaves][16 * OP];
  __shared__ float ml_lds[kPWaves][16][2];
  const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int G = Hq / Hkv, lane = threadIdx.x & 63, wave = wave_id();
  const int col = lane & 15, quad = lane >> 4;
  const Sequence sq = sequence_of(pg, b, T, room);
  if (nblk == 1) {  // no merge follows: the rows that are no tokens are written here
    const int first = sq.ok ? sq.count : 0;
    for (int e = threadIdx.x; e < (T - first) * G * D; e += 64 * kPWaves) {
      const int t = first + e / (G * D);
      o.out[(((size_t)b * T + t) * Hq + h * G) * D + e % (G * D)] = sq.ok ? 0 : kNanBits;
    }
  }
  const int total = sq.len + sq.count, key0 = c * BLK;
  if (!sq.ok || sq.count == 0 || key0 >= total) return;
  const int a0 = key0 + wave * ATOM;
  const bool active = a0 < total;

  // The pages of the atom's 16-key granules; one past the sequence's end repeats the first, one whose page is none
  // takes page 0, masked below.
  bf16x8_t kf[KT][KS];
  u32x4_t vf[PS * DT];
  uint32_t bad = 0;
  if (active) {
    const int32_t* row = pg.table + (size_t)b * pg.ld;
    const int P = 1 << pg.log2p;
    const uint16_t *kb[GR], *vb[GR];
#pragma unroll
    for (int j = 0; j < GR; ++j) {
      const int at = a0 + 16 * j < total ? a0 + 16 * j : a0;
      int page = row[at >> pg.log2p];
      if ((unsigned)page >= (unsigned)pg.n_pages) {
        page = 0;
        bad |= 1u << j;
      }
      const int in = at & (P - 1);
      kb[j] = pg.k + (int64_t)page * pg.k_stride + ((size_t)h * P + in) * D;
      vb[j] = pg.vt + (int64_t)page * pg.vt_stride + (size_t)h * D * P + in;
    }
    // K rows of tile kt in the order row r -> key 32(kt/2) + 8(r/4) + 4(kt%2) + r%4, so that a lane's scores are
    // the eight consecutive keys of its quad that P's operand wants.
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int kk = 8 * (col >> 2) + 4 * (kt & 1) + (col & 3);
      const uint16_t* kr = (col >= 8 ? kb[2 * (kt >> 1) + 1] : kb[2 * (kt >> 1)]) + (kk & 15) * D + quad * 8;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[kt][ks] = *reinterpret_cast<const bf16x8_t*>(kr + ks * 32);
    }
#pragma unroll
    for (int s = 0; s < PS; ++s) {
      const uint16_t* vr = (quad >= 2 ? vb[2 * s + 1] : vb[2 * s]) + (size_t)col * P + 8 * (quad & 1);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) vf[s * DT + dt] = *reinterpret_cast<const u32x4_t*>(vr + (size_t)dt * 16 * P);
    }
    // Slots past the sequence hold anything: their values are zeroed, for 0 * NaN is NaN.
    if (a0 + ATOM > total || bad) {
#pragma unroll
      for (int s = 0; s < PS; ++s) {
        int n = min(max(total - (a0 + 32 * s + 8 * quad), 0), 8);
        if ((bad >> (2 * s + (quad >> 1))) & 1) n = 0;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vf[s * DT + dt] = first_keys(vf[s * DT + dt], n);
      }
    }
  }
  // New tokens' values that are no numbers must not reach the rows before them.
  const bool odd = active && sq.count > 1 && a0 + ATOM > sq.len + 1 && any_not_finite(vf);

  const int rows = sq.count * G;
  const int nact = min(kPWaves, (total - key0 + ATOM - 1) / ATOM);
  const float sc = scale * kPLog2e;
  for (int r0 = 0; r0 < rows; r0 += 16) {
    const int n = min(16, rows - r0);
    if (active) {
      const int qr = r0 + min(col, n - 1);
      const int t = qr / G;
      const int last = col < n ? sq.len + t : -1;  // the last position this row sees
      const uint16_t* qp = q + (((size_t)b * T + t) * Hq + h * G + qr % G) * D + quad * 8;
      bf16x8_t qf[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8_t*>(qp + ks * 32);
      float s[KT][4];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) acc = mfma16x16x32(kf[kt][ks], qf[ks], acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[kt][i] = acc[i] * sc;
      }
      if (bad) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
          if ((bad >> (2 * (kt >> 1) + (quad >> 1))) & 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[kt][i] = __builtin_nanf("");
      }
      const int k0 = a0 + 8 * quad;
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (k0 + 32 * (kt >> 1) + 4 * (kt & 1) + i > last) s[kt][i] = -INFINITY;
          mx = fmaxf(mx, s[kt][i]);
        }
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mref = mx == -INFINITY ? 0.f : mx;
      // P as the sum of two bf16 terms (2^-17 of each weight; one term's 2^-9 would be as large as the output's own
      // rounding). The matrix cores wait for memory either way.
      u32x4_t hi[PS], lo[PS];
      float sum = 0.f;
#pragma unroll
      for (int ks = 0; ks < PS; ++ks)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int kt = 2 * ks + (w >> 1), i = 2 * (w & 1);
          const float p0 = __builtin_amdgcn_exp2f(s[kt][i] - mref), p1 = __builtin_amdgcn_exp2f(s[kt][i + 1] - mref);
          sum += p0;
          sum += p1;
          const uint32_t h0 = f32_to_bf16_bits(p0), h1 = f32_to_bf16_bits(p1);
          hi[ks][w] = h0 | (h1 << 16);
          lo[ks][w] = (uint32_t)f32_to_bf16_bits(p0 - bf16_bits_to_f32(h0)) |
                      ((uint32_t)f32_to_bf16_bits(p1 - bf16_bits_to_f32(h1)) << 16);
        }
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      f32x4_t acc[DT];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (!odd) {
#pragma unroll
        for (int ks = 0; ks < PS; ++ks)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const bf16x8_t v = __builtin_bit_cast(bf16x8_t, vf[ks * DT + dt]);
            acc[dt] = mfma16x16x32(v, __builtin_bit_cast(bf16x8_t, hi[ks]), acc[dt]);
            acc[dt] = mfma16x16x32(v, __builtin_bit_cast(bf16x8_t, lo[ks]), acc[dt]);
          }
      } else {  // token by token, each with the values that it sees
        const int t1 = (r0 + n - 1) / G;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          for (int tt = r0 / G; tt <= t1; ++tt) {
            f32x4_t one = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < PS; ++ks) {
              const int nk = min(max(sq.len + tt + 1 - (k0 + 32 * ks), 0), 8);
              const bf16x8_t v = __builtin_bit_cast(bf16x8_t, first_keys(vf[ks * DT + dt], nk));
              one = mfma16x16x32(v, __builtin_bit_cast(bf16x8_t, hi[ks]), one);
              one = mfma16x16x32(v, __builtin_bit_cast(bf16x8_t, lo[ks]), one);
            }
            if (tt == t) acc[dt] = one;
          }
      }
      if (col < n) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          *reinterpret_cast<f32x4_t*>(&o_lds[wave][col * OP + dt * 16 + quad * 4]) = acc[dt];
        if (quad == 0) {
          ml_lds[wave][col][0] = mx;
          ml_lds[wave][col][1] = sum;
        }
      }
    }
    __syncthreads();
    // Fold the atoms in order: thread e takes four dims of a row.
    for (int e = threadIdx.x; e < n * (D / 4); e += 64 * kPWaves) {
      const int r = e / (D / 4), d = (e % (D / 4)) * 4;
      float m = -INFINITY;
      for (int w = 0; w < nact; ++w) m = fmaxf(m, ml_lds[w][r][0]);
      const float mref = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < nact; ++w) {
        const float f = __builtin_amdgcn_exp2f(ml_lds[w][r][0] - mref);
        l = fmaf(f, ml_lds[w][r][1], l);
        const f32x4_t v = *reinterpret_cast<const f32x4_t*>(&o_lds[w][r * OP + d]);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(f, v[i], acc[i]);
      }
      const int qr = r0 + r;
      if (nblk == 1) {
        const size_t orow = (size_t)b * T + qr / G;
        const int head = h * G + qr % G;
        const uint16_t* gp = o.gate ? o.gate + (int64_t)orow * o.ldg + (int64_t)head * o.gs : nullptr;
        uint16_t* op = o.out + (orow * Hq + head) * D + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) op[i] = finished(acc[i], l, gp, d + i);
      } else {
        const size_t at = (((size_t)b * Hkv + h) * nblk + c) * (size_t)(T * G) + qr;
        *reinterpret_cast<f32x4_t*>(part_o + at * D + d) = acc;
        if (d == 0) {
          part_ml[2 * at] = m;
          part_ml[2 * at + 1] = l;
        }
      }
    }
    __syncthreads();
  }
}

// One workgroup per (query head, token, sequence): the row's blocks joined, wave w taking blocks w, w + 4, ..., the
// waves' sums then in order.
template <int D>
__global__ __launch_bounds__(64 * kPMergeWaves) void paged_merge_kernel(Pages pg, int T, int Hq, int Hkv, int room, int nblk,
                                                                        const float* __restrict__ part_o,
                                                                        const float* __restrict__ part_ml, Out o) {
  constexpr int E = D / 64;
  __shared__ float red[kPMergeWaves], suml[kPMergeWaves], sumo[kPMergeWaves][D];
  const int head = blockIdx.x, t = blockIdx.y, b = blockIdx.z, G = Hq / Hkv, h = head / G;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const Sequence sq = sequence_of(pg, b, T, room);
  const size_t orow = (size_t)b * T + t;
  uint16_t* op = o.out + (orow * Hq + head) * D;
  if (!sq.ok || t >= sq.count) {
    for (int d = threadIdx.x; d < D; d += 64 * kPMergeWaves) op[d] = sq.ok ? 0 : kNanBits;
    return;
  }
  const int nb = (sq.len + t) / paged_block(D) + 1;  // the blocks that this row sees
  const size_t base = ((size_t)b * Hkv + h) * nblk * (size_t)(T * G) + (size_t)t * G + head % G;
  const size_t step = (size_t)T * G;
  float m = -INFINITY;
  for (int c = threadIdx.x; c < nb; c += 64 * kPMergeWaves) m = fmaxf(m, part_ml[2 * (base + c * step)]);
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
  if (lane == 0) red[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPMergeWaves; ++w) m = fmaxf(m, red[w]);
  const float mref = m == -INFINITY ? 0.f : m;
  float l = 0.f, acc[E] = {};
  for (int c = wave; c < nb; c += kPMergeWaves) {
    const size_t at = base + c * step;
    const float f = __builtin_amdgcn_exp2f(part_ml[2 * at] - mref);
    l = fmaf(f, part_ml[2 * at + 1], l);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(f, part_o[at * D + lane + 64 * e], acc[e]);
  }
  if (lane == 0) suml[wave] = l;
#pragma unroll
  for (int e = 0; e < E; ++e) sumo[wave][lane + 64 * e] = acc[e];
  __syncthreads();
  const uint16_t* gp = o.gate ? o.gate + (int64_t)orow * o.ldg + (int64_t)head * o.gs : nullptr;
  for (int d = threadIdx.x; d < D; d += 64 * kPMergeWaves) {
    float lt = 0.f, ot = 0.f;
#pragma unroll
    for (int w = 0; w < kPMergeWaves; ++w) {
      lt += suml[w];
      ot += sumo[w][d];
    }
    op[d] = finished(ot, lt, gp, d);
  }
}

size_t paged_workspace(int B, int T, int Hq, int Hkv, int D, int keys) {
  const size_t nblk = ((size_t)keys + paged_block(D) - 1) / paged_block(D);
  if (nblk == 1) return 0;
  return (size_t)B * Hkv * nblk * T * (Hq / Hkv) * (D + 2) * sizeof(float);
}

bool head_dim_ok(int D) { return D == 64 || D == 128 || D == 256; }

// What both entry points ask of the cache; sets `pg`.
int check_pages(const skinny_paged_kv* kv, int B, int T, int Hq, Pages& pg, const char* what) {
  SKINNY_CHECK_ARG(kv && kv->lengths && kv->pages && kv->k_pages && kv->vt_pages, "%s: null pointer", what);
  SKINNY_CHECK_ARG(head_dim_ok(kv->head_dim), "%s: head dim %d unsupported (64, 128 or 256)", what, kv->head_dim);
  SKINNY_CHECK_ARG(kv->n_kv >= 1 && kv->n_kv <= 65535 && Hq >= kv->n_kv && Hq <= 65535 && Hq % kv->n_kv == 0,
                   "%s: Hq=%d must be a multiple of Hkv=%d", what, Hq, kv->n_kv);
  SKINNY_CHECK_ARG(B >= 1 && B <= 65535 && T >= 1 && T <= 65535, "%s: B=%d sequences of T=%d tokens (1 to 65535 each)",
                   what, B, T);
  const int P = kv->page;
  SKINNY_CHECK_ARG(P >= 16 && P <= 256 && (P & (P - 1)) == 0, "%s: page=%d slots (a power of two, 16 to 256)", what, P);
  SKINNY_CHECK_ARG(kv->n_pages >= 1 && kv->max_pages >= 1 && kv->ld_pages >= kv->max_pages &&
                       (int64_t)kv->max_pages * P <= (1 << 30),
                   "%s: n_pages=%d, max_pages=%d, ld_pages=%d", what, kv->n_pages, kv->max_pages, kv->ld_pages);
  const int64_t need = (int64_t)kv->n_kv * P * kv->head_dim;
  SKINNY_CHECK_ARG(kv->k_stride >= need && kv->vt_stride >= need && kv->k_stride % 8 == 0 && kv->vt_stride % 8 == 0,
                   "%s: page strides %lld, %lld (multiples of 8, at least Hkv*P*D=%lld)", what, (long long)kv->k_stride,
                   (long long)kv->vt_stride, (long long)need);
  SKINNY_CHECK_ARG(skinny_aligned(kv->k_pages, 16) && skinny_aligned(kv->vt_pages, 16) && skinny_aligned(kv->lengths, 4) &&
                       skinny_aligned(kv->counts, 4) && skinny_aligned(kv->pages, 4),
                   "%s: misaligned cache", what);
  pg = Pages{kv->lengths, kv->counts, kv->pages, kv->k_pages, kv->vt_pages, kv->k_stride, kv->vt_stride, kv->ld_pages,
             kv->n_pages, __builtin_ctz(P)};
  return SKINNY_OK;
}

template <int D>
int launch_paged_attention(const Pages& pg, const uint16_t* q, int B, int T, int Hq, int Hkv, int keys, float scale, float* ws,
                           const Out& o, hipStream_t s) {
  const int nblk = (keys + paged_block(D) - 1) / paged_block(D);
  const size_t parts = (size_t)B * Hkv * nblk * T * (Hq / Hkv);
  hipLaunchKernelGGL(paged_block_kernel<D>, dim3(nblk, Hkv, B), dim3(64 * kPWaves), 0, s, pg, q, T, Hq, Hkv, keys, scale, nblk,
                     ws, ws + parts * D, o);
  if (const int rc = skinny_check_launch("paged_attention")) return rc;
  if (nblk == 1) return SKINNY_OK;
  hipLaunchKernelGGL(paged_merge_kernel<D>, dim3(Hq, T, B), dim3(64 * kPMergeWaves), 0, s, pg, T, Hq, Hkv, keys, nblk, ws,
                     ws + parts * D, o);
  return skinny_check_launch("paged_attention merge");
}

}  // namespace

extern "C" int skinny_paged_store_bf16(const uint16_t* qkv, int ldq, int B, int T, int Hq, int q_stride, int k_offset,
                                       int v_offset, const uint16_t* q_norm, const uint16_t* k_norm, float eps,
                                       int rotary_dim, const float* rope_table, int rope_positions,
                                       const skinny_paged_kv* kv, uint16_t* q_out, void* stream) {
  Pages pg;
  if (const int rc = check_pages(kv, B, T, Hq, pg, "paged_store")) return rc;
  const int D = kv->head_dim, Hkv = kv->n_kv, room = kv->max_pages * kv->page;
  SKINNY_CHECK_ARG(qkv && rope_table && q_out, "paged_store: null pointer");
  SKINNY_CHECK_ARG(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= D,
                   "paged_store: rotary_dim=%d must be even, in [2, D=%d]", rotary_dim, D);
  SKINNY_CHECK_ARG(q_stride >= D && k_offset >= 0 && v_offset >= 0 && (int64_t)(Hq - 1) * q_stride + D <= ldq &&
                       (int64_t)k_offset + (int64_t)Hkv * D <= ldq && (int64_t)v_offset + (int64_t)Hkv * D <= ldq,
                   "paged_store: heads do not fit the q|k|v row of %d", ldq);
  SKINNY_CHECK_ARG(rope_positions >= room, "paged_store: RoPE table of %d positions, the pages hold %d", rope_positions, room);
  SKINNY_CHECK_ARG(skinny_aligned(qkv, 2) && skinny_aligned(rope_table, 8) && skinny_aligned(q_out, 16) &&
                       skinny_aligned(q_norm, 2) && skinny_aligned(k_norm, 2),
                   "paged_store: misaligned buffer");
  const dim3 grid(Hq + 2 * Hkv, T, B);
  const hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(64), 0, s, pg, qkv, ldq, T, Hq, Hkv, q_stride, k_offset, v_offset, q_norm, k_norm,
                       eps, rotary_dim, rope_table, room, q_out);
  };
  if (D == 64) go(paged_store_kernel<64>);
  else if (D == 128) go(paged_store_kernel<128>);
  else go(paged_store_kernel<256>);
  return skinny_check_launch("paged_store");
}

extern "C" size_t skinny_paged_attn_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int keys) {
  if (B < 1 || T < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || !head_dim_ok(D) || keys < 1 || (int64_t)T * (Hq / Hkv) > kPMaxRows)
    return 0;
  return paged_workspace(B, T, Hq, Hkv, D, keys);
}

extern "C" int skinny_paged_attention_bf16(const uint16_t* q, int B, int T, int Hq, const skinny_paged_kv* kv, int keys,
                                           float scale, const uint16_t* gate, int64_t ld_gate, int gate_stride,
                                           void* workspace, size_t workspace_bytes, uint16_t* out, void* stream) {
  Pages pg;
  if (const int rc = check_pages(kv, B, T, Hq, pg, "paged_attention")) return rc;
  const int D = kv->head_dim, Hkv = kv->n_kv;
  SKINNY_CHECK_ARG(q && out, "paged_attention: null pointer");
  SKINNY_CHECK_ARG((int64_t)T * (Hq / Hkv) <= kPMaxRows, "paged_attention: %lld query rows per kv head, at most %d",
                   (long long)T * (Hq / Hkv), kPMaxRows);
  SKINNY_CHECK_ARG(keys >= 1 && keys <= kv->max_pages * kv->page, "paged_attention: keys=%d, the pages hold %d", keys,
                   kv->max_pages * kv->page);
  SKINNY_CHECK_ARG(!gate || (gate_stride >= 0 && ld_gate >= 0),
                   "paged_attention: gate strides %lld, %d", (long long)ld_gate, gate_stride);
  SKINNY_CHECK_ARG(skinny_aligned(q, 16) && skinny_aligned(out, 16) && skinny_aligned(gate, 2) && skinny_aligned(workspace, 16),
                   "paged_attention: misaligned buffer");
  const size_t need = paged_workspace(B, T, Hq, Hkv, D, keys);
  SKINNY_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need), "paged_attention: workspace of %zu bytes, needs %zu",
                   workspace ? workspace_bytes : (size_t)0, need);
  const Out o{out, gate, ld_gate, gate_stride};
  float* ws = static_cast<float*>(workspace);
  const hipStream_t s = (hipStream_t)stream;
  if (D == 64) return launch_paged_attention<64>(pg, q, B, T, Hq, Hkv, keys, scale, ws, o, s);
  if (D == 128) return launch_paged_attention<128>(pg, q, B, T, Hq, Hkv, keys, scale, ws, o, s);
  return launch_paged_attention<256>(pg, q, B, T, Hq, Hkv, keys, scale, ws, o, s);
}
