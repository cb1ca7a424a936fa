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
#include <type_traits>
#include "paged.h"

using namespace paged;

namespace {

constexpr int kPMaxRuns = 65535;  // runs of a sequence: a grid's last index

// A block's keys, and the waves that share it: 64 KB of K and V for 128 and 256 dims, a wave's part of which is 64 registers.
__host__ __device__ constexpr int paged_block(int D) { return D == 256 ? 64 : 128; }
__host__ __device__ constexpr int paged_waves(int D) { return D == 64 ? 2 : 4; }
constexpr int kPQuad = 4;      // blocks joined left to right
constexpr int kPLanes = 8;     // running joins of groups in the merge
constexpr int kPGroup = 8;     // blocks whose quads are joined left to right

// ---------------------------------------------------------------------------------------------------------
// New rows into the cache. A wave takes 64 / (D / 8) query or key heads of a token, eight dims a lane; or 64 value dims of
// the tokens of 16 slots, a dim per lane, which it turns over in registers, so that they go out in 16-byte pieces. Bound by
// latency for few tokens and by memory for many.

// Granules of 16 slots that T tokens can touch, after the one that holds the first of them.
__host__ __device__ constexpr uint32_t granules_after_first(int T) { return (T + 14) / 16; }

// Eight bf16 at any even address.
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any_t __attribute__((ext_vector_type(4), aligned(8)));

struct StoreRows {
  const uint16_t* qkv;
  int ldq, qs, koff, voff;
  const uint16_t *qn, *kn;  // null: no norm
};

template <int D>
__device__ __forceinline__ void store_heads(const Pages& pg, const StoreRows& rows, int T, int Hq, int Hkv, float eps, int R,
                                            const float* __restrict__ rope, int room, uint16_t* __restrict__ q_out, int unit,
                                            float* __restrict__ lds) {
  constexpr int LPH = D / 8, HPW = 64 / LPH;
  const int lane = threadIdx.x & 63, t = blockIdx.y, b = blockIdx.z;
  const int head = unit * HPW + lane / LPH, d0 = lane % LPH * 8;
  const bool there = head < Hq + Hkv;
  const size_t r = (size_t)b * T + t;
  const bool query = head < Hq;
  u32x4_t x4 = {0, 0, 0, 0}, w4 = {0, 0, 0, 0};
  const uint16_t* norm = query ? rows.qn : rows.kn;
  if (there) {
    const size_t at = query ? head * (size_t)rows.qs : rows.koff + (size_t)(head - Hq) * D;
    x4 = *reinterpret_cast<const u32x4_any_t*>(rows.qkv + r * rows.ldq + at + d0);
    if (norm) w4 = *reinterpret_cast<const u32x4_any_t*>(norm + d0);
  }
  const Sequence sq = sequence_of(pg, b, T, room);
  const bool live = sq.ok && t < sq.count;
  const int pos = live ? sq.len + t : 0;
  const int page = live ? words(pg.table)[(size_t)b * pg.ld + (pos >> pg.log2p)] : -1;
  u32x4_t* qd = reinterpret_cast<u32x4_t*>(q_out + (r * Hq + head) * D + d0);
  if ((unsigned)page >= (unsigned)pg.n_pages) {  // no token, or nowhere to put it
    const uint32_t fill = sq.ok && t >= sq.count ? 0u : kNanBits * 0x10001u;
    if (query) *qd = u32x4_t{fill, fill, fill, fill};
    return;
  }
  const int half = R >> 1;
  const bool turns = d0 < R;
  // the table's entries of these dims: pair i = d, or d - half
  const float* cs = rope + ((size_t)pos * half) * 2;
  const bool whole = half % 8 == 0;  // eight dims turn together, with the eight of one other lane
  f32x4_t c4[4];
  if (whole && turns)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c4[i] = *reinterpret_cast<const f32x4_any_t*>(cs + 2 * (d0 < half ? d0 : d0 - half) + 4 * i);
  float x[8], ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = bf16_bits_to_f32(e & 1 ? x4[e >> 1] >> 16 : x4[e >> 1] & 0xffffu);
    ss = fmaf(x[e], x[e], ss);
  }
  if (rows.qn || rows.kn) {
    ss = dpp_add<0xB1>(ss);
    ss = dpp_add<0x4E>(ss);
    ss = dpp_add<0x141>(ss);
    if (LPH >= 16) ss = dpp_add<0x140>(ss);
    if (LPH >= 32) ss += __shfl_xor(ss, 16, 64);
    const float inv = rsqrtf(ss / (float)D + eps);
    if (norm)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= inv * bf16_bits_to_f32(e & 1 ? w4[e >> 1] >> 16 : w4[e >> 1] & 0xffffu);
  }
  // The pairs' other halves through LDS: [head][D], this wave's own.
  float* mine = lds + lane / LPH * D;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    *reinterpret_cast<f32x4_t*>(mine + d0 + 4 * i) = f32x4_t{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if (whole) {
    if (turns) {
      const float sign = d0 < half ? -1.f : 1.f;
      const float* other = mine + (d0 < half ? d0 + half : d0 - half);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * c4[e >> 1][2 * (e & 1)] + sign * other[e] * c4[e >> 1][2 * (e & 1) + 1];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = d0 + e;
      if (d < R) {
        const int i = d < half ? d : d - half;
        const float other = mine[d < half ? d + half : d - half];
        x[e] = x[e] * cs[2 * i] + (d < half ? -other : other) * cs[2 * i + 1];
      }
    }
  }
  u32x4_t y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = two_bf16(x[2 * i], x[2 * i + 1]);
  if (!there) return;
  const int slot = pos & ((1 << pg.log2p) - 1);
  if (query) *qd = y;
  else
    *reinterpret_cast<u32x4_t*>(pg.k + (int64_t)page * (int64_t)pg.k_stride +
                                (((size_t)(head - Hq) << pg.log2p) + slot) * D + d0) = y;
}

// 64 dims from `dim` on, of the value rows' Hkv * D, of the tokens in a granule's 16 slots: a dim per lane.
template <int D>
__device__ __forceinline__ void store_values(const Pages& pg, const StoreRows& rows, int T, int Hkv, int room, int granule,
                                             int dim) {
  const int lane = threadIdx.x & 63, b = blockIdx.z;
  if (dim >= Hkv * D) return;
  const Sequence sq = sequence_of(pg, b, T, room);
  if (!sq.ok || sq.count == 0) return;
  const int p0 = ((sq.len >> 4) + granule) << 4;  // the granule's first position
  if (p0 >= sq.len + sq.count) return;
  const int page = words(pg.table)[(size_t)b * pg.ld + (p0 >> pg.log2p)];
  if ((unsigned)page >= (unsigned)pg.n_pages) return;
  const int s0 = max(sq.len - p0, 0), s1 = min(sq.len + sq.count - p0, 16);  // its slots that are written
  const uint16_t* src = rows.qkv + ((int64_t)b * T + (p0 - sq.len)) * rows.ldq + rows.voff + dim + lane;
  const int P = 1 << pg.log2p;
  uint16_t* dst = pg.vt + (int64_t)page * (int64_t)pg.vt_stride + (size_t)(dim + lane) * P + (p0 & (P - 1));
  if (s1 - s0 == 1) {
    dst[s0] = src[(int64_t)s0 * rows.ldq];
    return;
  }
  // Pieces of eight slots, with what a piece's other slots hold: stores of single values wait for each other where they
  // meet in a line (8 tokens of 16 sequences, 4 heads of 256 dims: 11 us so).
  u32x4_t old[2];
  uint32_t v[16];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    old[i] = u32x4_t{0, 0, 0, 0};
    if (s0 < 8 * i + 8 && s1 > 8 * i && (s0 > 8 * i || s1 < 8 * i + 8)) old[i] = *reinterpret_cast<const u32x4_t*>(dst + 8 * i);
  }
#pragma unroll
  for (int s = 0; s < 16; ++s) v[s] = src[(int64_t)min(max(s, s0), s1 - 1) * rows.ldq];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (s0 >= 8 * i + 8 || s1 <= 8 * i) continue;
    u32x4_t w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int s = 8 * i + 2 * k;
      const uint32_t lo = s < s0 || s >= s1 ? old[i][k] & 0xffffu : v[s];
      const uint32_t hi = s + 1 < s0 || s + 1 >= s1 ? old[i][k] >> 16 : v[s + 1];
      w[k] = lo | hi << 16;
    }
    *reinterpret_cast<u32x4_t*>(dst + 8 * i) = w;
  }
}

// Grid (workgroups of four head units, then of values; tokens; sequences). A sequence's value workgroups, `value_groups` (of 256
// dims) for each granule that T tokens can touch, are dealt over the tokens. The first extent is odd, for the eight dies take
// workgroups in turn and the values' are the slow ones. Two prompts of up to 1501 tokens: 18.4 us; 22.0 with an even extent,
// 19.8 with a granule's workgroups at every token, most of which have none.
template <int D>
__global__ __launch_bounds__(256) void paged_store_kernel(Pages pg, StoreRows rows, int T, int Hq, int Hkv, float eps, int R,
                                                          const float* __restrict__ rope, int room, int head_groups,
                                                          uint32_t value_groups, uint16_t* __restrict__ q_out) {
  __shared__ __attribute__((aligned(16))) float lds[4][512];
  const int wave = wave_id();
  if ((int)blockIdx.x < head_groups)
    store_heads<D>(pg, rows, T, Hq, Hkv, eps, R, rope, room, q_out, (int)blockIdx.x * 4 + wave, lds[wave]);
  else {
    const uint32_t i = ((int)blockIdx.x - head_groups) * T + (int)blockIdx.y, granule = i / value_groups;
    if (granule <= granules_after_first(T))
      store_values<D>(pg, rows, T, Hkv, room, granule, ((i - granule * value_groups) * 4 + wave) * 64);
  }
}

// ---------------------------------------------------------------------------------------------------------
// Attention. A workgroup takes a run of blocks of keys of one sequence and kv head. In a block each wave scores its share of
// the keys (S^T = K Q^T, the K rows straight from memory into matrix-core operands); the row maxima and then the weights P go
// through LDS, and each wave forms its share of the dims over all the block's keys (O^T = V^T P^T). So K and V are read once,
// by one wave each, and no output is summed across waves. As soon as a block's scores (outputs) are formed, its K (V)
// registers take the next block's loads, which are in flight through the rest of the block.
//
// What bounds it is memory, if the instructions of a block (64 KB of K and V for 128 dims) stay few: everything that only a
// block at the sequence's end, or one with a missing page, needs stands behind one branch, and addresses are formed in
// scalars once per page. One token of 4 sequences of 65536 keys, 8 heads of 128 dims: 180 us, 5.9 TB/s; of 32 sequences of up
// to 2048 keys 31 us, 4.5 TB/s.
//
// Blocks are joined left to right in quads, quads in groups of kPGroup blocks, groups by the merge. All are cut at fixed
// positions of the sequence, and keys that a row does not see add exact zeros, so a row's bits depend on its own sequence
// and position alone: not on the batch, on T, on who joins the blocks, or on where the pages lie.

// W tiles of 16 query rows; a call of more rows per kv head than 32 (kHalves) takes two workgroups a run, the second
// of which finds K and V in the caches. by_g: 65536 / G rounded up, G = Hq / Hkv. GS: keys of a block that share a page: the
// page size where that is 16 or 32, else 64.
//
// Grid (heads, sequences, runs): the eight dies take workgroups in turn, so neighbours are heads, whose work is alike, and
// the runs that a sequence turns out not to have come last, of little cost. With the runs first, 32 sequences of 1023
// keys took, in groups, 44 us a call for a bound of 1032 keys and 61 for one of 4112 (runs of eight: a die each); so 31
// and 33. 64 of up to 1000: 42 and 38.
template <int D, int W, int GS, bool kHalves>
__global__ __launch_bounds__(64 * paged_waves(D), 2) void paged_block_kernel(Pages pg, const uint16_t* __restrict__ q, int T,
                                                                             int G, int by_g, int Hq, int Hkv, int room,
                                                                             float scale, int span, int slots,
                                                                             float* __restrict__ part_o,
                                                                             float* __restrict__ part_ml, Out o) {
  constexpr int BLK = paged_block(D), WAVES = paged_waves(D);
  constexpr int KT = BLK / 16 / WAVES, KS = D / 32;           // a wave's 16-key tiles; dim steps of a score
  constexpr int ST = BLK / 32, NG = BLK / GS;                 // a block's 32-key steps and pages
  constexpr int KG = KT * 16 > GS ? KT * 16 / GS : 1;         // pages of a wave's keys
  constexpr int DW = D / 16 / WAVES;                          // a wave's 16-dim tiles
  constexpr bool kKept = W == 1 && D != 256;                  // the queries stay in registers
  constexpr int QP = D + 8;                                   // else their pitch in LDS
  __shared__ u32x4_t p_lds[W][2][ST][64];
  __shared__ __attribute__((aligned(16))) float m_lds[W * 16][WAVES], l_lds[W * 16][WAVES];
  __shared__ __attribute__((aligned(16))) uint16_t q_lds[kKept ? 8 : W * 16 * QP];
  const bool second = kHalves && (int)blockIdx.x >= Hkv;
  const int h = second ? blockIdx.x - Hkv : blockIdx.x, b = blockIdx.y, slot = blockIdx.z;
  const int row0 = second ? 16 * W : 0;  // of the rows per kv head
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int col = lane & 15, quad = lane >> 4;
  const int c0 = slot * span;
  // The queries, the first block's pages and the lengths are asked for at once.
  constexpr int QN = kKept ? KS : (W * 16 * (D / 8) + 64 * WAVES - 1) / (64 * WAVES);
  auto token = [&](int r) { return r * by_g >> 16; };  // of row r, which is head r - token * G
  auto q_row = [&](int r) { return q + (uint32_t)((token(r) * (Hq - G) + r) * D); };
  q += ((size_t)b * T * Hq + (size_t)h * G) * D;
  u32x4_t qr[QN];
#pragma unroll
  for (int i = 0; i < QN; ++i) {
    const int e = threadIdx.x + i * 64 * WAVES;
    const int r = kKept ? col : e / (D / 8), d = kKept ? i * 32 + quad * 8 : e % (D / 8) * 8;
    qr[i] = *reinterpret_cast<const u32x4_t*>(q_row(min(row0 + r, T * G - 1)) + d);
  }
  // A block's pages (idk: those of the wave's own keys).
  const words_t table = words(pg.table + (size_t)b * pg.ld);
  const int log2p = GS == 16 ? 4 : GS == 32 ? 5 : pg.log2p;
  const int P = 1 << log2p;
  const int own = wave * (KT * 16) / GS;
  int ids[NG], idk[KG];
  auto find = [&](int c) {
    if ((c + 1) * BLK <= pg.max_pages << log2p) {
#pragma unroll
      for (int g = 0; g < NG; ++g) ids[g] = GS < 64 ? table[c * NG + g] : table[(c * BLK + g * GS) >> log2p];
#pragma unroll
      for (int g = 0; g < KG; ++g) idk[g] = GS < 64 ? table[c * NG + own + g] : table[(c * BLK + (own + g) * GS) >> log2p];
    } else {
#pragma unroll
      for (int g = 0; g < NG; ++g) ids[g] = table[min((c * BLK + g * GS) >> log2p, pg.max_pages - 1)];
#pragma unroll
      for (int g = 0; g < KG; ++g) idk[g] = table[min((c * BLK + (own + g) * GS) >> log2p, pg.max_pages - 1)];
    }
  };
  find(c0);
  const Sequence sq = sequence_of(pg, b, T, room);
  if (slots == 1 && row0 == 0) {  // no merge follows: the rows that are no tokens are written here
    const int first = sq.ok ? sq.count : 0;
    for (int e = threadIdx.x; e < (T - first) * G * D; e += 64 * WAVES) {
      const int t = first + e / (G * D);
      o.out[(((size_t)b * T + t) * Hq + h * G) * D + e % (G * D)] = sq.ok ? 0 : kNanBits;
    }
  }
  const int total = sq.len + sq.count;
  if (!sq.ok || sq.count == 0 || c0 * BLK >= total) return;
  const int c1 = min(c0 + span, (total + BLK - 1) / BLK);
  const int rows = sq.count * G;
  if (row0 >= rows) return;
  const float sc = scale * kPLog2e;
  // Pages past the sequence become the block's first; one that is none becomes page 0, its bit set.
  uint32_t bad = 0;
  auto settle = [&](int c) {
    uint32_t top = 0, none = 0;
#pragma unroll
    for (int g = 0; g < NG; ++g) top = max(top, (uint32_t)ids[g]);
    if ((c + 1) * BLK > total || top >= (uint32_t)pg.n_pages) {
      auto fit = [&](int id, int g) { return c * BLK + g * GS < total ? id : ids[0]; };
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        const int id = fit(idk[g], own + g);
        idk[g] = (unsigned)id < (unsigned)pg.n_pages ? id : 0;
      }
#pragma unroll
      for (int g = NG - 1; g >= 0; --g) {
        const int id = fit(ids[g], g);
        const bool there = (unsigned)id < (unsigned)pg.n_pages;
        ids[g] = there ? id : 0;
        none |= there ? 0u : 1u << g;
      }
    }
    return none;
  };
  bf16x8_t kf[KT][KS];
  u32x4_t vf[ST][DW];
  const uint16_t* k_head = pg.k + (size_t)h * P * D;
  const uint16_t* v_head = pg.vt + ((size_t)h * D + 16 * DW * wave) * P;
  const uint32_t k_lane = col * D + quad * 8;
  auto load_k = [&](int c) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int in = (c * BLK + 16 * (wave * KT + kt)) & (P - 1);
      const uint16_t* kr = k_head + ((uint64_t)(uint32_t)idk[kt * 16 / GS] * pg.k_stride + in * D);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[kt][ks] = *reinterpret_cast<const bf16x8_t*>(kr + (k_lane + ks * 32));
    }
  };
  // V^T rows: dims 16DW wave + 16dt + col, keys 32s + 8quad + 0..7 of the block. Loaded past the caches' retention where no
  // other workgroup wants them, a dim tile's steps one after the other, so that the two halves of a line of 64 keys are asked
  // for together. 64 sequences of 4000 keys of 128 dims with pages of 16 / 64 slots: 193 / 197 us with ordinary loads, 184 /
  // 190 so, K's loads alike 201 / 202; in 64-dim heads 107 / 108, 90 / 98. With two workgroups a run 328 / 338 as it is, 361 /
  // 401 past the caches.
  const uint32_t v_lane = col * P + 8 * (GS == 16 ? quad & 1 : quad);
  auto load_v = [&](int c) {
#pragma unroll
    for (int dt = 0; dt < DW; ++dt)
#pragma unroll
      for (int s = 0; s < ST; ++s) {
        auto base = [&](int i) {
          const int key = 32 * s + 16 * i;
          const int in = (GS < 64 ? key : c * BLK + key) & (P - 1);
          return v_head + ((uint64_t)(uint32_t)ids[key / GS] * pg.vt_stride + in);
        };
        const uint16_t* vr = base(0);
        if constexpr (GS == 16) vr = quad >= 2 ? base(1) : vr;
        const u32x4_t* at = reinterpret_cast<const u32x4_t*>(vr + (v_lane + dt * 16 * P));
        vf[s][dt] = kHalves ? *at : __builtin_nontemporal_load(at);
      }
  };

  bad = settle(c0);
  load_k(c0);
  load_v(c0);
  bf16x8_t qf[KS];
  if constexpr (kKept) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = __builtin_bit_cast(bf16x8_t, qr[ks]);
  } else {
#pragma unroll
    for (int i = 0; i < QN; ++i) {
      const int e = threadIdx.x + i * 64 * WAVES;
      if (e < W * 16 * (D / 8)) *reinterpret_cast<u32x4_t*>(&q_lds[e / (D / 8) * QP + e % (D / 8) * 8]) = qr[i];
    }
    lds_barrier();
  }

  // The quad's and the group's maximum (log2 units) and sum of this lane's row of every tile, and its outputs.
  float am[W], al[W], gm[W], gl[W];
  f32x4_t ao[W][DW], go[W][DW];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    am[w] = gm[w] = -INFINITY;
    al[w] = gl[w] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DW; ++dt) ao[w][dt] = go[w][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  for (int c = c0; c < c1; ++c) {
    const int key0 = c * BLK;
    const bool more = c + 1 < c1;
    const bool edge = key0 + BLK > sq.len + 1 || bad;  // some row does not see, or may not read, some key
    if (more) find(c + 1);
    float s[W][KT][4];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w && row0 + 16 * w >= rows) continue;
      if constexpr (!kKept) {
        const uint16_t* qp = &q_lds[(16 * w + col) * QP + quad * 8];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8_t*>(qp + ks * 32);
      }
      f32x4_t acc[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) acc[kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) acc[kt] = mfma16x16x32(kf[kt][ks], qf[ks], acc[kt]);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[w][kt][i] = acc[kt][i];
    }
    uint32_t bad_next = 0;
    if (more) {
      bad_next = settle(c + 1);
      load_k(c + 1);
    }
    if (edge) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int r = row0 + 16 * w + col;
        const int last = (r < rows ? sq.len + token(r) : -1) - (key0 + 16 * wave * KT + 4 * quad);  // of the lane's keys
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const bool none = (bad >> (own + kt * 16 / GS)) & 1;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[w][kt][i] = 16 * kt + i > last ? -INFINITY : none ? __builtin_nanf("") : s[w][kt][i];
        }
      }
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w && row0 + 16 * w >= rows) continue;
      float mx = s[w][0][0];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[w][kt][i]);
      mx = quads_max(mx);
      if (quad == 0) m_lds[16 * w + col][wave] = mx;
    }
    lds_barrier();
    float mx[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w && row0 + 16 * w >= rows) continue;
      float m = m_lds[16 * w + col][0];
#pragma unroll
      for (int v = 1; v < WAVES; ++v) m = fmaxf(m, m_lds[16 * w + col][v]);
      mx[w] = m * sc;
      const float ref = mx[w] == -INFINITY ? 0.f : mx[w];  // finite scores too, if the scale takes all of them there
      // P as the sum of two bf16 terms (2^-17 of each weight; one term's 2^-9 would be as large as the output's own
      // rounding).
      float sum = 0.f;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        u32x2_t hi, lo;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(s[w][kt][2 * v], sc, -ref));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(s[w][kt][2 * v + 1], sc, -ref));
          sum += p0;
          sum += p1;
          hi[v] = two_bf16(p0, p1);
          lo[v] = two_bf16(p0 - __uint_as_float(hi[v] << 16), p1 - __uint_as_float(hi[v] & 0xffff0000u));
        }
        // keys 16g + 4quad .. + 3: half of the piece that lane (col, quad g, quad / 2) of step g / 2 takes
        const int g = wave * KT + kt, at = col + 16 * (2 * (g & 1) + (quad >> 1));
        reinterpret_cast<u32x2_t*>(&p_lds[w][0][g >> 1][at])[quad & 1] = hi;
        reinterpret_cast<u32x2_t*>(&p_lds[w][1][g >> 1][at])[quad & 1] = lo;
      }
      sum = quads_sum(sum);
      if (quad == 0) l_lds[16 * w + col][wave] = sum;
    }
    lds_barrier();
    f32x4_t acc[W][DW];
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int dt = 0; dt < DW; ++dt) acc[w][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // Slots past the sequence hold anything: their values are zeroed, for 0 * NaN is NaN. So are new tokens' values that
    // are no numbers, which no earlier row may meet: the outputs that see one begin as NaN instead.
    if (edge) {
      uint32_t odd[DW] = {};  // bits 4st + v and 16 + 4st + v: the halves of word v of the step's piece are no numbers
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        int n = min(max(total - (key0 + 32 * st + 8 * quad), 0), 8);
        if ((bad >> (GS == 16 ? 2 * st + (quad >> 1) : 32 * st / GS)) & 1) n = 0;
#pragma unroll
        for (int dt = 0; dt < DW; ++dt) {
          vf[st][dt] = first_keys(vf[st][dt], n);
          if (sq.count == 1) continue;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            // an exponent of all ones carries into the half's top bit
            const uint32_t no = ((vf[st][dt][v] & 0x7f807f80u) + 0x00800080u) >> 15 & 0x00010001u;
            vf[st][dt][v] &= ~(no * 0xffffu);
            odd[dt] |= no << (4 * st + v);
          }
          asm volatile("" : "+v"(vf[st][dt]), "+v"(odd[dt]));  // piece by piece: interleaved, they take twice the registers
        }
      }
      uint32_t any = odd[0];
#pragma unroll
      for (int dt = 1; dt < DW; ++dt) any |= odd[dt];
      if (__any(any != 0)) {
        // How many of them each output's row sees: a product of the odd values' and the seen keys' ones.
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int r = row0 + 16 * w + col, seen = (r < rows ? sq.len + token(r) + 1 : 0) - (key0 + 8 * quad);
#pragma unroll
          for (int dt = 0; dt < DW; ++dt) {
#pragma unroll 1
            for (int st = 0; st < ST; ++st) {
              u32x4_t a, k = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
              for (int v = 0; v < 4; ++v) a[v] = (odd[dt] >> (4 * st + v) & 0x00010001u) * 0x3f80u;
              k = first_keys(k, min(max(seen - 32 * st, 0), 8));
              acc[w][dt] = mfma16x16x32(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, k), acc[w][dt]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[w][dt][i] = acc[w][dt][i] > 0.f ? __builtin_nanf("") : 0.f;
          }
        }
      }
    }
    float l[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w && row0 + 16 * w >= rows) continue;
      l[w] = l_lds[16 * w + col][0];
#pragma unroll
      for (int v = 1; v < WAVES; ++v) l[w] += l_lds[16 * w + col][v];
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const bf16x8_t hi = __builtin_bit_cast(bf16x8_t, p_lds[w][0][st][lane]);
        const bf16x8_t lo = __builtin_bit_cast(bf16x8_t, p_lds[w][1][st][lane]);
#pragma unroll
        for (int dt = 0; dt < DW; ++dt) acc[w][dt] = mfma16x16x32(__builtin_bit_cast(bf16x8_t, vf[st][dt]), hi, acc[w][dt]);
#pragma unroll
        for (int dt = 0; dt < DW; ++dt) acc[w][dt] = mfma16x16x32(__builtin_bit_cast(bf16x8_t, vf[st][dt]), lo, acc[w][dt]);
      }
    }
    if (more) load_v(c + 1);
    bad = bad_next;
    const bool end = !more || (c + 1) % kPQuad == 0;  // of the quad
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w && row0 + 16 * w >= rows) continue;
      const Join j = join(am[w], al[w], mx[w], l[w]);
#pragma unroll
      for (int dt = 0; dt < DW; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) ao[w][dt][i] = fmaf(acc[w][dt][i], j.part, ao[w][dt][i] * j.before);
      if (!end) continue;
      const Join g = join(gm[w], gl[w], am[w], al[w]);
#pragma unroll
      for (int dt = 0; dt < DW; ++dt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) go[w][dt][i] = fmaf(ao[w][dt][i], g.part, go[w][dt][i] * g.before);
        ao[w][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
      am[w] = -INFINITY;
      al[w] = 0.f;
    }
  }
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int r = row0 + 16 * w + col, d0 = wave * 16 * DW + quad * 4;
    if (r >= rows) continue;
    if (slots > 1) {  // a part, for the merge
      const size_t at = (((size_t)b * Hkv + h) * slots + slot) * (size_t)(T * G) + r;
#pragma unroll
      for (int dt = 0; dt < DW; ++dt) *reinterpret_cast<f32x4_t*>(part_o + at * D + d0 + dt * 16) = go[w][dt];
      if (wave == 0 && quad == 0) reinterpret_cast<float2*>(part_ml)[at] = float2{gm[w], gl[w]};
      continue;
    }
    const int t = token(r), head = h * G + r - t * G;
    const size_t orow = (size_t)b * T + t;
    const uint16_t* gp = o.gate ? o.gate + (int64_t)orow * o.ldg + (int64_t)head * o.gs : nullptr;
    const float inv = 1.f / gl[w];
#pragma unroll
    for (int dt = 0; dt < DW; ++dt) {
      u32x2_t two;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int d = d0 + dt * 16 + 2 * i;
        two[i] = finished(go[w][dt][2 * i], inv, gp, gp ? gp[d] : 0) |
                 (uint32_t)finished(go[w][dt][2 * i + 1], inv, gp, gp ? gp[d + 1] : 0) << 16;
      }
      *reinterpret_cast<u32x2_t*>(o.out + (orow * Hq + head) * D + d0 + dt * 16) = two;
    }
  }
}

// The rows' groups joined: group g in order onto lane g % kPLanes, then the lanes in order. A row is one wave's, holding all
// lanes, or (kSplit) a workgroup's with a wave for each. A slot of the workspace is kSlot blocks: a group, or a quad or a
// block, joined to its group here as the block kernel would. Bound by latency: a launch and two round trips, 4 to 5.5 us.
template <int D, int kSlot, bool kSplit>
__global__ __launch_bounds__(kSplit ? 64 * kPLanes : 256) void paged_merge_kernel(Pages pg, int T, int Hq, int G, int Hkv,
                                                                                  int room, int slots,
                                                                                  const float* __restrict__ part_o,
                                                                                  const float* __restrict__ part_ml, Out o) {
  constexpr int E = D / 64, L = kSplit ? 1 : kPLanes;      // lanes of groups that a wave holds
  constexpr int N = kPGroup / kSlot;                       // slots of a group
  constexpr int UN = 8 / (L * N) > 1 ? 8 / (L * N) : 1;    // rounds of groups loaded at once
  __shared__ __attribute__((aligned(16))) float sum[kSplit ? kPLanes : 1][kSplit ? D : 1];
  __shared__ float ml[kSplit ? kPLanes : 1][2];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int head = kSplit ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave, t = blockIdx.y, b = blockIdx.z;
  if (head >= Hq) return;
  const WorkIndex in = work_index(head, G);  // the kv head, and the head's place in its group
  const size_t step = (size_t)T * G;
  const size_t base = ((size_t)b * Hkv + in.quot) * slots * step + (size_t)t * G + in.rem;
  typedef float dims_t __attribute__((ext_vector_type(E)));  // a lane's: E * lane on
  float pm[UN][L][N], pl[UN][L][N];
  dims_t po[UN][L][N];
  auto load = [&](int g0) {
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int i = 0; i < L; ++i)
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const size_t at = base + (size_t)min((g0 + kPLanes * u + i) * N + n, slots - 1) * step;
          const float2 two = reinterpret_cast<const float2*>(part_ml)[at];
          pm[u][i][n] = two.x;
          pl[u][i][n] = two.y;
          po[u][i][n] = *reinterpret_cast<const dims_t*>(part_o + at * D + E * lane);
        }
  };
  int g0 = kSplit ? wave : 0;
  load(g0);  // beside the lengths and the gate: slots that this row turns out not to have are not used
  const size_t orow = (size_t)b * T + t;
  const uint16_t* gp = o.gate ? o.gate + (int64_t)orow * o.ldg + (int64_t)head * o.gs : nullptr;
  uint32_t gate[E] = {};
  if (gp) {
    if constexpr (kSplit) gate[0] = gp[threadIdx.x % D];
    else
#pragma unroll
      for (int e = 0; e < E; ++e) gate[e] = gp[E * lane + e];
  }
  const Sequence sq = sequence_of(pg, b, T, room);
  uint16_t* op = o.out + (orow * Hq + head) * D;
  if (!sq.ok || t >= sq.count) {
    if (!kSplit || wave == 0)
      for (int d = lane; d < D; d += 64) op[d] = sq.ok ? 0 : kNanBits;
    return;
  }
  // the blocks, slots and groups that this row sees
  const int nb = (sq.len + t) / paged_block(D) + 1, ns = (nb + kSlot - 1) / kSlot, ng = (nb + kPGroup - 1) / kPGroup;
  float m[L], l[L];
  dims_t acc[L];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    acc[i] = dims_t(0.f);
  }
  while (g0 < ng) {
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int g = g0 + kPLanes * u + i;
        if (g >= ng) continue;
        float gm = -INFINITY, gl = 0.f, am = -INFINITY, al = 0.f;
        dims_t go(0.f), ao(0.f);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (g * N + n < ns) {
            const Join j = join(am, al, pm[u][i][n], pl[u][i][n]);
#pragma unroll
            for (int e = 0; e < E; ++e) ao[e] = fmaf(po[u][i][n][e], j.part, ao[e] * j.before);
          }
          if ((n + 1) * kSlot % kPQuad == 0) {
            const Join j = join(gm, gl, am, al);
#pragma unroll
            for (int e = 0; e < E; ++e) {
              go[e] = fmaf(ao[e], j.part, go[e] * j.before);
              ao[e] = 0.f;
            }
            am = -INFINITY;
            al = 0.f;
          }
        }
        const Join j = join(m[i], l[i], gm, gl);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[i][e] = fmaf(go[e], j.part, acc[i][e] * j.before);
      }
    g0 += kPLanes * UN;
    if (g0 < ng) load(g0);
  }
  if constexpr (!kSplit) {
    float rm = -INFINITY, rl = 0.f;
    dims_t ro(0.f);
#pragma unroll
    for (int i = 0; i < kPLanes; ++i) {
      const Join j = join(rm, rl, m[i], l[i]);
#pragma unroll
      for (int e = 0; e < E; ++e) ro[e] = fmaf(acc[i][e], j.part, ro[e] * j.before);
    }
    const float inv = 1.f / rl;
    typedef uint16_t out_t __attribute__((ext_vector_type(E)));
    out_t y;
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = finished(ro[e], inv, gp, gate[e]);
    *reinterpret_cast<out_t*>(op + E * lane) = y;
  } else {
    if (lane == 0) {
      ml[wave][0] = m[0];
      ml[wave][1] = l[0];
    }
    *reinterpret_cast<dims_t*>(&sum[wave][E * lane]) = acc[0];
    __syncthreads();
    if (const int d = threadIdx.x; d < D) {
      float rm = -INFINITY, rl = 0.f, ro = 0.f;
#pragma unroll
      for (int w = 0; w < kPLanes; ++w) {
        const Join j = join(rm, rl, ml[w][0], ml[w][1]);
        ro = fmaf(sum[w][d], j.part, ro * j.before);
      }
      op[d] = finished(ro, 1.f / rl, gp, gate[0]);
    }
  }
}

int paged_blocks(int keys, int D) { return (keys + paged_block(D) - 1) / paged_block(D); }

// Blocks per workgroup: one, a quad, or a group. Single blocks are the most parallel; the more a workgroup takes, the
// fewer parts are written and read again (of 32 rows of 128 dims a quarter of a block's own bytes) and the longer its loads
// stay in flight from block to block, but it takes enough of them to fill the card, also where sequences end early; one
// part a sequence needs no merge. Measured, us a call by blocks / quads / groups, 4 query heads per kv head, B x keys:
// one token, 8 heads of 128 dims: 1 x 2048 (136 blocks) 10.0 / 16.1 / 25.3, 1 x 8192 (520) 16.1 / 17.4 / 26.6, 4 x 4000
// (1024) 20.1 / 19.4 / 28.1, 16 x 2000 (2048) 30.5 / 29.5 / 30.7, 32 of up to 2048 (4352) 41.5 / 38.2 / 46.2, 16 x 8000
// (8064) 103 / 92 / 91, 64 x 4000 (16384) 238 / 204 / 193; in one part, 64 x 300 30.2 / 21.3, 64 x 1000 58 / 52 / 48, 16 x
// 500 14.2 / 14.6. Eight tokens: 4 x 1000 (256) 14.9 / 18.7 / 25.3, 1 x 8192 (520) 22.3 / 18.9 / 28.6, 16 x 2000 54 / 36 /
// 35, 12 of up to 4000 51 / 34 / 43 and 52 / 41 / 47, 12 x 4000 70 / 51 / 53, 32 of up to 2048 78 / 53 / 53, 48 of
// up to 2000 (6144) 105 / 66 / 61; six tokens, 256 dims, 16 of up to 4000 (4032) 75 / 55 / 50. One token, 4 heads of 256
// dims: 1 x 8192 (516) 17.1 / 17.3 / 25.5, 8 x 4000 (2016) 30.8 / 29.0 / 28.4, 32 x 2000 (4096) 59 / 52 / 50; 9 of up to
// 5003, 3 tokens (2880) 37 / 37 / 44. 8 heads of 64 dims: 1 x 8192 11.5 / 13.7 / 20.9, 16 x 2000 19.3 / 18.2 / 22.9, 64 x
// 4000 92 / 93 / 101, 64 x 8000 (32256) 207 / 190 / 189. 64 dims have no threshold of their own, so that the rule takes groups
// for the last but one, the slowest of the three there. The blocks are those of the host's bound: short sequences under a
// large bound are cut as long ones are (32 of up to 2048 keys: 35 us, under a bound 8 times as large 45).
int paged_span(int B, int Hkv, int nblk, int rows, int D) {
  const int64_t heads = (int64_t)B * Hkv, all = heads * nblk;
  const bool heavy = rows > 16;
  if (all >= (D == 256 ? (heavy ? 3000 : 4096) : heavy ? 4096 : 8192) || (nblk <= kPGroup && nblk > kPQuad && heads >= 256))
    return kPGroup;
  return all >= (heavy ? 400 : D == 256 ? 512 : 1536) || (nblk <= kPQuad && heads >= 128) ? kPQuad : 1;
}

int paged_slots(int nblk, int span) { return (nblk + span - 1) / span; }

size_t paged_workspace(int B, int T, int Hq, int Hkv, int D, int keys) {
  const int nblk = paged_blocks(keys, D), slots = paged_slots(nblk, paged_span(B, Hkv, nblk, T * (Hq / Hkv), D));
  if (slots == 1) return 0;
  return (size_t)B * Hkv * slots * T * (Hq / Hkv) * (D + 2) * sizeof(float);
}

template <int D>
int launch_paged_attention(const Pages& pg, const uint16_t* q, int B, int T, int Hq, int Hkv, int keys, float scale, float* ws,
                           const Out& o, hipStream_t s) {
  const int G = Hq / Hkv, rows = T * G;
  const int nblk = paged_blocks(keys, D), span = paged_span(B, Hkv, nblk, rows, D), slots = paged_slots(nblk, span);
  float* ml = ws + (size_t)B * Hkv * slots * rows * D;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(rows > 32 ? 2 * Hkv : Hkv, B, slots), dim3(64 * paged_waves(D)), 0, s, pg, q, T, G,
                       65535 / G + 1, Hq, Hkv, keys, scale, span, slots, ws, ml, o);
  };
  auto page = [&](auto w, auto h) {
    constexpr int W = decltype(w)::value;
    constexpr bool kHalves = decltype(h)::value;
    if (pg.log2p == 4) go(paged_block_kernel<D, W, 16, kHalves>);
    else if (pg.log2p == 5) go(paged_block_kernel<D, W, 32, kHalves>);
    else go(paged_block_kernel<D, W, 64, kHalves>);
  };
  if (rows <= 16) page(std::integral_constant<int, 1>{}, std::false_type{});
  else if (rows <= 32) page(std::integral_constant<int, 2>{}, std::false_type{});
  else page(std::integral_constant<int, 2>{}, std::true_type{});
  if (const int rc = skinny_check_launch("paged_attention")) return rc;
  if (slots == 1) return SKINNY_OK;
  const int groups = (nblk + kPGroup - 1) / kPGroup;
  // eight waves a row where the rows alone would not fill the card, and always for blocks
  const bool split = span == 1 || (int64_t)B * T * Hq <= (groups > 8 ? 1024 : 512);
  auto merge = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(split ? Hq : (Hq + 3) / 4, T, B), dim3(split ? 64 * kPLanes : 256), 0, s, pg, T, Hq, G, Hkv,
                       keys, slots, ws, ml, o);
  };
  if (span == 1) merge(paged_merge_kernel<D, 1, true>);
  else if (span == kPQuad && split) merge(paged_merge_kernel<D, kPQuad, true>);
  else if (span == kPQuad) merge(paged_merge_kernel<D, kPQuad, false>);
  else if (split) merge(paged_merge_kernel<D, kPGroup, true>);
  else merge(paged_merge_kernel<D, kPGroup, false>);
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
  const int heads = 64 / (D / 8) * 4, groups = (Hq + Hkv + heads - 1) / heads;  // query and key heads of a workgroup
  const int values = (Hkv * (D / 64) + 3) / 4;
  const StoreRows rows{qkv, ldq, q_stride, k_offset, v_offset, q_norm, k_norm};
  const hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((groups + (values * (granules_after_first(T) + 1) + T - 1) / T) | 1, T, B), dim3(256), 0, s,
                       pg, rows, T, Hq, Hkv, eps, rotary_dim, rope_table, room, groups, values, q_out);
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
  const int nblk = paged_blocks(keys, D);
  SKINNY_CHECK_ARG(paged_slots(nblk, paged_span(B, Hkv, nblk, T * (Hq / Hkv), D)) <= kPMaxRuns,
                   "paged_attention: keys=%d, at most %d", keys, kPMaxRuns * kPGroup * paged_block(D));
  SKINNY_CHECK_ARG(scale > 0.f && scale <= 1e38f, "paged_attention: scale=%g must be positive", (double)scale);
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
