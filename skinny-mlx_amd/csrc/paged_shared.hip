// Attention of sequences that begin with one prefix, in a cache in pages: the prefix's keys and values are read once for
// the whole batch, whose query rows then make matrix products of them, where paged.hip reads each sequence's own.
//
// No reference counterpart: the reference decodes one sequence (skinny_mlx/spec.py:98-156). Arithmetic of a layer as at
// spec.py:24-29 (causal GQA attention, optionally output * sigmoid(gate)).
//
// A row's softmax over [the prefix; its own keys] is joined from parts: runs of the prefix's keys, formed for all rows by
// workgroups, and runs of a sequence's own keys, formed for its rows by single waves. Both are workgroups of one launch, so that
// the first ones' products and the others' loads share the card; a second launch joins them.
#include <type_traits>
#include <cmath>
#include "paged.h"

using namespace paged;

namespace {

struct Prefix {
  const int32_t* length;
  const int32_t* pages;
  int max_pages, room;
};

// The keys that the call may read, -1 where the length cannot be.
__device__ __forceinline__ int prefix_length(const Prefix& p) {
  const int n = words(p.length)[0];
  return n >= 0 && n <= p.room ? n : -1;
}

// A workgroup of NW waves takes 16 * RT * NW / KW query rows of a kv head (every sequence's, one after the other) and a run of
// the prefix: NW / KW groups of 16 * RT rows, in each of which KW waves share a tile's keys. A tile of keys is staged in LDS as
// the matrix cores' operands and read by all the row groups; the next tile's loads are in flight meanwhile. Four lanes in a row
// load 64 bytes of a K (V) row at once (a row a lane: 3 % slower, 64 sequences of 500 behind 32768 tokens) and
// put them where the lanes that want them read without bank conflicts: the 16 rows of an operand's quad q in order row ^ 4q.
// Scores are formed transposed, S^T = K Q^T, with the K rows of a 32-key step taken so that a lane holds eight consecutive keys of
// one query row, which is the operand that O^T = V^T P^T wants: P never leaves its lane.
//
// P is the sum of two bf16 terms, 2^-16 of a weight, as in paged.hip and for the own keys. (One term, 2^-8, is half of the matrix
// products with V; it left results 2.0e-3 to 2.3e-3 off where their own rounding is 1.65e-3, and 64 sequences of 1000 behind 32768
// tokens took 94 us for 97.) The running maximum is raised only where a score passes it by 2^8: until then weights up to 2^8
// are as exact, and the outputs need no rescaling.
//
// Bound by the matrix cores, LDS reads and the exponentials, which take about as long each, where rows are many (256 of 8 heads of
// 128 dims: each 32768 keys more 47 us, 730 TFLOP/s of the two products), by loads where they are few.
template <int D>
struct Shape {
  static constexpr int KS = D / 32;   // dim steps of a score
  static constexpr int DT = D / 16;   // dim tiles of an output
};

constexpr float kLag = 8.f;

// Keys of a tile: 64 KB of K and V for 128 and 256 dims, whose loads are in flight through a tile's products.
__host__ __device__ constexpr int tile_keys(int D) { return D == 256 ? 64 : 128; }

template <int D, int RT, int KW, int NW>
__host__ __device__ constexpr int prefix_lds() {
  const int tiles = 2 * 2 * tile_keys(D) * D * 2;                                   // K and V, two buffers
  const int join = KW > 1 ? NW * 16 * RT * (D + 4) * 4 + NW * 16 * RT * 2 * 4 : 0;  // the waves' outputs, maxima and sums
  return tiles > join ? tiles : join;
}

// What both roles are given.
struct Rows {
  const uint16_t* q;
  int B, T, G, Hq, Hkv;
  float scale;
  float *part_o, *part_ml;
};

template <int D, int RT, int KW, int NW>
__device__ __forceinline__ void prefix_run(const Pages& pg, const Prefix& px, const Rows& x, int h, int row_block, int slot, int span) {
  constexpr int KS = Shape<D>::KS, DT = Shape<D>::DT, TK = tile_keys(D);
  constexpr int ST = TK / 32;        // 32-key steps of a tile
  constexpr int NF = TK * D / 512;   // 1 KB operands of K, and of V, in a tile
  constexpr int FW = NF / NW;        // a wave's share of them, all of one step
  extern __shared__ u32x4_t lds[];   // [buffer][K operands, V operands][lane]
  const int G = x.G, TG = x.T * G, Hq = x.Hq, rows = x.B * TG;
  const int lane = threadIdx.x & 63, wave = wave_id(), col = lane & 15, quad = lane >> 4;
  const int kw = wave % KW, row0 = (row_block * (NW / KW) + wave / KW) * (16 * RT);
  // The pages of a wave's step of a tile: its first sixteen keys' and the others'. Asked for a tile before they are used.
  const words_t table = words(px.pages);
  const int step = 32 * (wave * ST / NW);  // of the tile
  int id[2];
  auto find = [&](int key0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) id[i] = table[min((key0 + step + 16 * i) >> pg.log2p, px.max_pages - 1)];
  };
  const int begin = slot * span;
  find(begin);
  const int len = prefix_length(px);
  const int end = min(begin + span, len);
  if (begin >= end) return;
  const float sc = x.scale * kPLog2e;
  // a flat row's sequence and row of that sequence's T * G
  auto row_of = [&](int r, int& b, int& in) {
    b = r / TG;
    in = r - b * TG;
  };
  const int P = 1 << pg.log2p;
  const uint16_t* k_head = pg.k + (size_t)h * P * D;
  const uint16_t* v_head = pg.vt + (size_t)h * D * P;
  u32x4_t kr[FW], vr[FW];
  bool bad = false;  // a page of the run that is none: every row of it is NaN
  // Operand f of a tile's K: step f / (2 KS), half a of its keys, dims 32 ks on. Row r of the half's product is key
  // 8 (r / 4) + 4a + r % 4 of the step. Of its V: step f / DT, dims 16 dt on.
  const int lrow = lane >> 2, lquad = lane & 3;
  const uint32_t k_lane = (8 * (lrow >> 2) + (lrow & 3)) * D + lquad * 8, v_lane = lrow * P + 8 * lquad;
  const int put = lquad * 16 + (lrow ^ 4 * lquad), get = quad * 16 + (col ^ 4 * quad);
  int tail = 0;  // of the loaded tile: the lane's V pieces' keys, where some are past the prefix
  bool edge = false;
  auto load = [&](int key0) {
    const int first = key0 + step;
    uint64_t kp[2], vp[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool ok = (unsigned)id[i] < (unsigned)pg.n_pages;
      bad |= !ok && first + 16 * i < len;
      const uint64_t page = ok ? (uint32_t)id[i] : 0u;
      // keys of a page of 16 begin at its first slot; larger pages hold the whole step
      const int in = (first & (P - 1)) - (P == 16 ? 16 * i : 0);
      kp[i] = page * pg.k_stride + (int64_t)in * D;
      vp[i] = page * pg.vt_stride + (int64_t)in;
    }
    const uint16_t* ka = k_head + (lrow >= 8 ? kp[1] : kp[0]);
    const uint16_t* va = v_head + (lquad >= 2 ? vp[1] : vp[0]);
#pragma unroll
    for (int i = 0; i < FW; ++i) {
      const int f = (wave * FW) % (2 * KS) + i;  // (a multiple of 2 KS if FW is)
      const int a = FW >= 2 * KS ? i / KS : f / KS, ks = FW >= KS ? i % KS : f % KS;
      kr[i] = *reinterpret_cast<const u32x4_t*>(ka + (k_lane + (uint32_t)(4 * a * D + ks * 32)));
    }
#pragma unroll
    for (int i = 0; i < FW; ++i) {
      const int dt = FW >= DT ? i : (wave * FW) % DT + i;
      vr[i] = *reinterpret_cast<const u32x4_t*>(va + (v_lane + (uint32_t)(dt * 16 * P)));
    }
    edge = first + 32 > len;
    tail = min(max(len - first - 8 * lquad, 0), 8);
  };
  auto stage = [&](int buf) {
    u32x4_t* to = lds + (size_t)buf * 2 * NF * 64 + wave * FW * 64 + put;
    if (edge) {  // slots past the prefix hold anything, and 0 * NaN is NaN
#pragma unroll
      for (int i = 0; i < FW; ++i) vr[i] = first_keys(vr[i], tail);
    }
#pragma unroll
    for (int i = 0; i < FW; ++i) {
      to[i * 64] = kr[i];
      to[(NF + i) * 64] = vr[i];
    }
  };
  load(begin);
  bf16x8_t qf[RT][KS];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int b, in;
    row_of(min(row0 + 16 * rt + col, rows - 1), b, in);
    const int t = in / G;
    const uint16_t* qp = x.q + (((size_t)b * x.T + t) * Hq + h * G + in - t * G) * D + quad * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[rt][ks] = *reinterpret_cast<const bf16x8_t*>(qp + ks * 32);
  }
  float m[RT];
  float sum[RT];  // of this lane's weights of a row
  f32x4_t o[RT][DT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    sum[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  if (begin + TK < end) find(begin + TK);
  stage(0);
  lds_barrier();
  constexpr int SW = ST / KW;  // a wave's steps of a tile
  const int steps = (end - begin + TK - 1) / TK * SW;
  // Scores of step `at`, past the run's end -inf.
  auto scores = [&](int at, f32x4_t (&acc)[RT][2]) {
    const int s = at % SW * KW + kw, tile = at / SW;
    const u32x4_t* kt = lds + (size_t)(tile & 1) * 2 * NF * 64 + s * (2 * KS * 64) + get;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) acc[rt][0] = acc[rt][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16x8_t kf = __builtin_bit_cast(bf16x8_t, kt[(a * KS + ks) * 64]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][a] = mfma16x16x32(kf, qf[rt][ks], acc[rt][a]);
      }
    const int left = end - (begin + tile * TK + 32 * s);
    if (left < 32) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (8 * quad + e >= left) acc[rt][e >> 2][e & 3] = -INFINITY;
    }
  };
  int at = 0, loaded = 0;
  bool fresh = false;  // the maximum has been raised for this very step
  for (;;) {
    // Steps that need no new maximum. (Its raise, which scales the outputs, stands outside this loop: on a branch inside it, the
    // compiler keeps the outputs in other registers, and moves all of them in every step that does not take it.)
    while (at < steps) {
      const int tile = at / SW;
      const bool more = begin + (tile + 1) * TK < end;
      if (loaded == tile && more) {
        load(begin + (tile + 1) * TK);
        if (begin + (tile + 2) * TK < end) find(begin + (tile + 2) * TK);
        loaded = tile + 1;
      }
      f32x4_t acc[RT][2];
      scores(at, acc);
      float t[RT][8];  // over the running maximum, in log2 units
      bool up = false;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float ref = m[rt] == -INFINITY ? 0.f : m[rt];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[rt][e] = fmaf(acc[rt][e >> 2][e & 3], sc, -ref);
        const float top = fmaxf(fmaxf(fmaxf(t[rt][0], t[rt][1]), fmaxf(t[rt][2], t[rt][3])),
                                fmaxf(fmaxf(t[rt][4], t[rt][5]), fmaxf(t[rt][6], t[rt][7])));
        up |= top > (m[rt] == -INFINITY ? -INFINITY : kLag);
      }
      if (!fresh && __any(up)) break;
      fresh = false;
      bf16x8_t hi[RT], lo[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        u32x4_t h, l;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float p0 = __builtin_amdgcn_exp2f(t[rt][2 * w]), p1 = __builtin_amdgcn_exp2f(t[rt][2 * w + 1]);
          sum[rt] += p0;
          sum[rt] += p1;
          h[w] = two_bf16(p0, p1);
          l[w] = two_bf16(p0 - __uint_as_float(h[w] << 16), p1 - __uint_as_float(h[w] & 0xffff0000u));
        }
        hi[rt] = __builtin_bit_cast(bf16x8_t, h);
        lo[rt] = __builtin_bit_cast(bf16x8_t, l);
      }
      const u32x4_t* vt = lds + ((size_t)(tile & 1) * 2 + 1) * NF * 64 + (at % SW * KW + kw) * (DT * 64) + get;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, vt[dt * 64]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          o[rt][dt] = mfma16x16x32(vf, hi[rt], o[rt][dt]);
          o[rt][dt] = mfma16x16x32(vf, lo[rt], o[rt][dt]);
        }
      }
      if (++at % SW == 0) {
        if (more) stage((tile + 1) & 1);
        lds_barrier();
      }
    }
    if (at == steps) break;
    // Only of the rows that pass theirs: when another row, maybe of another sequence, raises its own is nothing to a row's bits.
    f32x4_t acc[RT][2];
    scores(at, acc);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float top = acc[rt][0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, acc[rt][e >> 2][e & 3]);
      top = quads_max(top);
      const bool none = m[rt] == -INFINITY, up = fmaf(top, sc, none ? 0.f : -m[rt]) > (none ? -INFINITY : kLag);
      const float nm = up ? top * sc : m[rt], f = up ? __builtin_amdgcn_exp2f(m[rt] - nm) : 1.f;
      m[rt] = nm;
      sum[rt] *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[rt][dt][i] *= f;
    }
    fresh = true;
  }
  // A page that was none, met by any wave.
  int* flag = reinterpret_cast<int*>(lds);
  if (threadIdx.x == 0) *flag = 0;
  lds_barrier();
  if (bad) *flag = 1;
  lds_barrier();
  const bool none = *flag != 0;
  lds_barrier();
  float l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) l[rt] = none ? __builtin_nanf("") : quads_sum(sum[rt]);
  const size_t part0 = ((size_t)slot * x.Hkv + h) * rows;  // parts: [run][kv head][row]
  if constexpr (KW == 1) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + 16 * rt + col;
      if (r >= rows) continue;
      const size_t at = part0 + r;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(x.part_o + at * D + dt * 16 + quad * 4) = o[rt][dt];
      if (quad == 0) reinterpret_cast<float2*>(x.part_ml)[at] = float2{m[rt], l[rt]};
    }
  } else {
    // The KW waves of a row group joined in their order.
    float* out = reinterpret_cast<float*>(lds);                       // [wave][16 RT][D + 4]
    float2* ml = reinterpret_cast<float2*>(out + NW * 16 * RT * (D + 4));  // [wave][16 RT]
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float* mine = out + ((size_t)wave * 16 * RT + 16 * rt + col) * (D + 4);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(mine + dt * 16 + quad * 4) = o[rt][dt];
      if (quad == 0) ml[wave * 16 * RT + 16 * rt + col] = float2{m[rt], l[rt]};
    }
    __syncthreads();
    const int group = wave / KW;
    for (int i = kw * 64 + lane; i < 16 * RT * (D / 4); i += KW * 64) {
      const int in = i / (D / 4), d = i % (D / 4) * 4, r = row0 + in;
      if (r >= rows) continue;
      float rm = -INFINITY, rl = 0.f;
      f32x4_t ro = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const int at = (group * KW + w) * 16 * RT + in;
        const float2 one = ml[at];
        const f32x4_t v = *reinterpret_cast<const f32x4_t*>(out + (size_t)at * (D + 4) + d);
        const Join j = join(rm, rl, one.x, one.y);
#pragma unroll
        for (int e = 0; e < 4; ++e) ro[e] = fmaf(v[e], j.part, ro[e] * j.before);
      }
      const size_t at = part0 + r;
      *reinterpret_cast<f32x4_t*>(x.part_o + at * D + d) = ro;
      if (d == 0) reinterpret_cast<float2*>(x.part_ml)[at] = float2{rm, rl};
    }
  }
}

// A wave takes a run of a sequence's own keys for 16 of its query rows of a kv head, 32 keys a step. Four lanes in
// a row load 64 bytes of a K (V) row at once, and the wave turns them into the matrix cores' operands through LDS of its own; as
// soon as a step's K (V) is there, its registers take the next one's loads. Bound by memory: 64 sequences of 1000 tokens, 262 MB,
// in 52 us. (Loaded as operands, a row a lane, 54; and 16 rows of 256 dims are left no registers.)
template <int D>
__device__ __forceinline__ void own_run(const Pages& pg, const Rows& x, int b, int h, int tile, int run, int runs, int run_keys, int room) {
  constexpr int KS = Shape<D>::KS, DT = Shape<D>::DT, CH = DT < 8 ? DT : 8;  // (CH: operands staged at a time)
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int begin = run * run_keys;
  const words_t table = words(pg.table + (size_t)b * pg.ld);
  int id[2];  // the pages of a step's first sixteen keys and of the others
  auto find = [&](int key0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) id[i] = table[min((key0 + 16 * i) >> pg.log2p, pg.max_pages - 1)];
  };
  find(begin);
  const Sequence sq = sequence_of(pg, b, x.T, room);
  const int total = sq.len + sq.count, rows = sq.count * x.G;
  if (!sq.ok || begin >= total || 16 * tile >= rows) return;
  const int end = min(begin + run_keys, total);
  const int r = 16 * tile + col, t = r / x.G;
  const int last = r < rows ? sq.len + t : -1;  // the last key that this lane's row sees
  extern __shared__ u32x4_t lds[];  // D = 256: the wave's queries, which no register is left for
  constexpr bool kFar = D == 256;
  const uint32_t area = wave_id() * (kFar ? CH + KS : CH) * 64;
  uint32_t mine = area + CH * 64 + lane;
  bf16x8_t qf[kFar ? 1 : KS];
  {
    const int in = min(r, rows - 1), token = in / x.G;
    const uint16_t* qp = x.q + (((size_t)b * x.T + token) * x.Hq + h * x.G + in - token * x.G) * D + quad * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (kFar) lds[mine + ks * 64] = *reinterpret_cast<const u32x4_t*>(qp + ks * 32);
      else qf[ks] = *reinterpret_cast<const bf16x8_t*>(qp + ks * 32);
    }
  }
  const int P = 1 << pg.log2p;
  const uint16_t* k_head = pg.k + (size_t)h * P * D;
  const uint16_t* v_head = pg.vt + (size_t)h * D * P;
  const int lrow = lane >> 2, lquad = lane & 3;  // of an operand, as it is loaded
  const uint32_t k_lane = (8 * (lrow >> 2) + (lrow & 3)) * D + lquad * 8, v_lane = lrow * P + 8 * lquad;
  const uint32_t put = area + lquad * 16 + (lrow ^ 4 * lquad), get = area + quad * 16 + (col ^ 4 * quad);
  u32x4_t kr[DT], vr[DT];
  // Operands c CH on of the step's K or V to LDS (an area of 16 D words a wave at most), where every lane's reads before are done:
  // a wave's go in their order.
  auto stage = [&](const u32x4_t (&of)[DT], int c) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < CH; ++i) lds[put + i * 64] = of[c * CH + i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  auto there = [&](int i) { return (unsigned)id[i] < (unsigned)pg.n_pages; };
  auto slot_of = [&](int key0, int i) { return (key0 & (P - 1)) - (P == 16 ? 16 * i : 0); };
  auto load_k = [&](int key0) {
    uint64_t at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) at[i] = (there(i) ? (uint32_t)id[i] : 0u) * (uint64_t)pg.k_stride + (int64_t)slot_of(key0, i) * D;
    const uint16_t* p = k_head + (lrow >= 8 ? at[1] : at[0]);
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kr[a * KS + ks] = *reinterpret_cast<const u32x4_t*>(p + (k_lane + (uint32_t)(4 * a * D + ks * 32)));
  };
  auto load_v = [&](int key0) {
    uint64_t at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) at[i] = (there(i) ? (uint32_t)id[i] : 0u) * (uint64_t)pg.vt_stride + (int64_t)slot_of(key0, i);
    const uint16_t* p = v_head + (lquad >= 2 ? at[1] : at[0]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) vr[dt] = *reinterpret_cast<const u32x4_t*>(p + (v_lane + (uint32_t)(dt * 16 * P)));
  };
  uint32_t bad = 0, bad_next = 0;  // halves of the step on a page that is none
  auto missing = [&](int key0) { return (!there(0) && key0 < total ? 1u : 0u) | (!there(1) && key0 + 16 < total ? 2u : 0u); };
  load_k(begin);
  load_v(begin);
  bad = missing(begin);
  if (begin + 32 < end) find(begin + 32);
  const float sc = x.scale * kPLog2e;
  float m = -INFINITY, l = 0.f;
  f32x4_t o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int key0 = begin; key0 < end; key0 += 32) {
    const bool more = key0 + 32 < end;
    const bool edge = key0 + 32 > sq.len + 1 || bad;  // some row does not see, or may not read, some key
    f32x4_t acc[2] = {};
    if (kFar) asm volatile("" : "+v"(mine));  // (read anew in every step)
#pragma unroll
    for (int c = 0; c < DT / CH; ++c) {
      stage(kr, c);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int a = (c * CH + i) / KS, ks = (c * CH + i) % KS;
        const bf16x8_t one = kFar ? __builtin_bit_cast(bf16x8_t, lds[mine + ks * 64]) : qf[kFar ? 0 : ks];
        acc[a] = mfma16x16x32(__builtin_bit_cast(bf16x8_t, lds[get + i * 64]), one, acc[a]);
      }
    }
    if (more) {
      bad_next = missing(key0 + 32);
      load_k(key0 + 32);
    }
    float s[8];  // of keys 8 quad + e
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = acc[e >> 2][e & 3];
    if (edge) {
      const bool none = bad >> (quad >> 1) & 1;
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = key0 + 8 * quad + e > last ? -INFINITY : none ? __builtin_nanf("") : s[e];
    }
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, s[e]);
    const float nm = fmaxf(m, quads_max(top) * sc), ref = nm == -INFINITY ? 0.f : nm, f = __builtin_amdgcn_exp2f(m - ref);
    m = nm;
    l *= f;
    u32x4_t hi, lo;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[2 * w], sc, -ref)), p1 = __builtin_amdgcn_exp2f(fmaf(s[2 * w + 1], sc, -ref));
      l += p0;
      l += p1;
      hi[w] = two_bf16(p0, p1);
      lo[w] = two_bf16(p0 - __uint_as_float(hi[w] << 16), p1 - __uint_as_float(hi[w] & 0xffff0000u));
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[dt][i] *= f;
    bool odd = false;
    if (edge) {
      // Slots past the sequence hold anything: zeroed, for 0 * NaN is NaN. So are new tokens' values that are no numbers, which no
      // earlier row may meet: the outputs that see one become NaN instead, by a product of the odd values' and the seen keys' ones.
      const int n = (bad >> (lquad >> 1)) & 1 ? 0 : min(max(total - (key0 + 8 * lquad), 0), 8);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) vr[dt] = first_keys(vr[dt], n);
      odd = sq.count > 1 && any_not_finite(vr);
    }
#pragma unroll
    for (int c = 0; c < DT / CH; ++c) {
      stage(vr, c);
      if (odd) {
        const u32x4_t one = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
        const bf16x8_t seen = __builtin_bit_cast(bf16x8_t, first_keys(one, min(max(last + 1 - (key0 + 8 * quad), 0), 8)));
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          u32x4_t v = lds[get + i * 64], is;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t no = ((v[w] & 0x7f807f80u) + 0x00800080u) >> 15 & 0x00010001u;  // exponents of all ones
            v[w] &= ~(no * 0xffffu);
            is[w] = no * 0x3f80u;
          }
          lds[get + i * 64] = v;
          const f32x4_t met = mfma16x16x32(__builtin_bit_cast(bf16x8_t, is), seen, f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c * CH + i][e] = met[e] > 0.f ? __builtin_nanf("") : o[c * CH + i][e];
        }
      }
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, lds[get + i * 64]);
        o[c * CH + i] = mfma16x16x32(vf, __builtin_bit_cast(bf16x8_t, hi), o[c * CH + i]);
        o[c * CH + i] = mfma16x16x32(vf, __builtin_bit_cast(bf16x8_t, lo), o[c * CH + i]);
      }
    }
    if (more) {
      load_v(key0 + 32);
      if (key0 + 64 < end) find(key0 + 64);
    }
    bad = bad_next;
  }
  l = quads_sum(l);
  if (r >= rows) return;
  // parts: [sequence][kv head][run][row of its T * G]
  const size_t at = (((size_t)b * x.Hkv + h) * runs + run) * (size_t)(x.T * x.G) + r;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(x.part_o + at * D + dt * 16 + quad * 4) = o[dt];
  if (quad == 0) reinterpret_cast<float2*>(x.part_ml)[at] = float2{m, l};
}

// The prefix's workgroups first (the eight dies take them in turn), then the own keys' waves, the runs that a sequence turns out
// not to have last.
template <int D, int RT, int KW, int NW>
__global__ __launch_bounds__(64 * NW, NW / 4) void shared_parts_kernel(Pages pg, Prefix px, Rows x, int row_blocks, int span, int front,
                                                                       int tiles, int runs, int run_keys, int room, float* own_o,
                                                                       float* own_ml) {
  const int i = blockIdx.x;
  if (i < front) {
    // a head's run (`unit`) by all its blocks of rows on one die, whose cache then reads it once (12 sequences of 4 tokens behind
    // 5003, 192 rows of 256 dims: 34.7 -> 32.9 us)
    const int units = front / row_blocks, dies = units % 8 == 0 ? 8 : 1, block = i / dies % row_blocks;
    const int unit = i / dies / row_blocks * dies + i % dies;
    prefix_run<D, RT, KW, NW>(pg, px, x, unit % x.Hkv, block, unit / x.Hkv, span);
  } else {
    uint32_t unit = __builtin_amdgcn_readfirstlane((uint32_t)(i - front) * NW + wave_id());
    const uint32_t tile = unit % tiles;
    unit /= tiles;
    const uint32_t h = unit % x.Hkv;
    unit /= x.Hkv;
    const uint32_t b = unit % x.B, run = unit / x.B;
    if ((int)run >= runs) return;
    x.part_o = own_o;
    x.part_ml = own_ml;
    own_run<D>(pg, x, b, h, tile, run, runs, run_keys, room);
  }
}

// How many times `of` goes into n >= 1, the rest counted.
__host__ __device__ constexpr int times(int n, int of) { return (n - 1) / of + 1; }

// The parts of a row joined: those of the prefix, then those of its own keys, part i by wave i % W of the row's W, the waves in
// order. Bound by latency for few rows, by the parts' bytes for many (2048 rows of 18 parts 6.4 us).
template <int D, int W>
__global__ __launch_bounds__(256) void shared_merge_kernel(Pages pg, Prefix px, int T, int Hq, int G, int Hkv,
                                                                            int room, int span, int own_keys, int slots,
                                                                            size_t first, const float* __restrict__ part_o,
                                                                            const float* __restrict__ part_ml, Out o) {
  constexpr int E = D / 64, UN = 8;
  typedef float dims_t __attribute__((ext_vector_type(E)));
  typedef uint16_t out_t __attribute__((ext_vector_type(E)));
  __shared__ __attribute__((aligned(16))) float sum[W][W > 1 ? D : 4];
  __shared__ float2 ml[W];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int head = W > 1 ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave, t = blockIdx.y, b = blockIdx.z;
  if (head >= Hq) return;
  const int w = W > 1 ? wave : 0;
  const Sequence sq = sequence_of(pg, b, T, room);
  const int len = prefix_length(px);
  const size_t orow = (size_t)b * T + t;
  out_t* op = reinterpret_cast<out_t*>(o.out + (orow * Hq + head) * D) + lane;
  if (!sq.ok || len < 0 || t >= sq.count) {
    const bool padding = sq.ok && t >= sq.count;
    if (w == 0) *op = out_t(padding ? (uint16_t)0 : kNanBits);
    return;
  }
  const int np = len ? times(len, span) : 0, n = np + (sq.len + t) / own_keys + 1;  // parts of the prefix; and of its own keys
  // parts of the prefix [run][kv head][row], from `first` on those of the own keys [sequence][kv head][run][row of its T * G]
  const int h = head / G;
  const size_t TG = (size_t)T * G, in = (size_t)t * G + head % G;
  const size_t rows = (size_t)gridDim.z * TG, front = h * rows + b * TG + in, own = first + ((size_t)b * Hkv + h) * slots * TG + in;
  float rm = -INFINITY, rl = 0.f;
  dims_t ro(0.f);
  for (int i0 = w; i0 < n; i0 += W * UN) {
    float2 x[UN];
    dims_t v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int i = min(i0 + u * W, n - 1);
      const size_t at = i < np ? front + (size_t)i * Hkv * rows : own + (size_t)(i - np) * TG;
      x[u] = reinterpret_cast<const float2*>(part_ml)[at];
      v[u] = *reinterpret_cast<const dims_t*>(part_o + at * D + E * lane);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (i0 + u * W >= n) continue;
      const Join j = join(rm, rl, x[u].x, x[u].y);
#pragma unroll
      for (int e = 0; e < E; ++e) ro[e] = fmaf(v[u][e], j.part, ro[e] * j.before);
    }
  }
  if constexpr (W > 1) {
    *reinterpret_cast<dims_t*>(&sum[w][E * lane]) = ro;
    if (lane == 0) ml[w] = float2{rm, rl};
    __syncthreads();
    if (w > 0) return;
#pragma unroll
    for (int i = 1; i < W; ++i) {
      const dims_t v = *reinterpret_cast<const dims_t*>(&sum[i][E * lane]);
      const Join j = join(rm, rl, ml[i].x, ml[i].y);
#pragma unroll
      for (int e = 0; e < E; ++e) ro[e] = fmaf(v[e], j.part, ro[e] * j.before);
    }
  }
  const uint16_t* gp = o.gate ? o.gate + (int64_t)orow * o.ldg + (int64_t)head * o.gs + E * lane : nullptr;
  const float inv = 1.f / rl;
  out_t y;
#pragma unroll
  for (int e = 0; e < E; ++e) y[e] = finished(ro[e], inv, gp, gp ? gp[e] : 0);
  *op = y;
}

// How a call is cut. The prefix: row tiles a wave, waves that share a tile's keys, keys of a run (`span`) and runs (`slots`). A
// sequence's own keys: 16-row tiles of its rows, keys of a run, runs.
struct Cut {
  int rt, kw, waves, row_blocks, span, slots;
  int tiles, own_keys, own_runs;
};

// The form of the prefix's kernel by the query rows of a kv head: few rows want the tile's keys dealt to many waves, many rows few
// reads of a tile. Behind 20000 tokens, us a call, (waves, row tiles, waves that share the keys):
//   8 heads of 128 dims:   (4, 1, 4) (8, 1, 4) (8, 2, 4) (8, 2, 2) (8, 2, 1)     4 heads of 256:  (4, 1, 2) (8, 1, 2) (8, 1, 1)
//            16 rows          23.2      23.4      27.1      34.8      47.0                           27.1      29.8      34.7
//            32               28.7      23.8      27.9      35.7      47.0                           27.7      31.1      36.6
//            64               44.5      31.3      29.1      36.7      47.9                           39.0      33.1      38.9
//           128               72.8      49.1      40.2      41.4      51.6                           55.5      47.4      46.5
//           256              146.0      87.8      67.0      65.2      63.0                          108.0      71.5      70.8
//   8 heads of 64 dims:
//            16 rows          17.8      17.5      18.4      23.1      32.0
//            32               20.7      17.0      18.8      24.0      32.4
//            64               29.8      21.1      20.3      24.8      33.1
//           128               47.0      32.5      30.7      28.7      35.0
//           256               81.4      48.9      46.2      42.5      42.0
void set_form(Cut& c, int rows, int D) {
  if (D == 256) {
    c.waves = rows > 32 ? 8 : 4;
    c.rt = 1;
    c.kw = rows > 64 ? 1 : 2;
  } else {
    c.waves = rows > 16 ? 8 : 4;
    c.rt = rows > 32 ? 2 : 1;
    c.kw = rows > 128 ? 1 : rows > 64 ? 2 : 4;
  }
}

// The runs. A CU holds one workgroup (of those of 64 dims and 16-row waves two, on which the cut does not count), so the card is
// shared out: so many workgroups to the prefix that those left over are done with the own keys in the same time. What a CU does, by
// the figures that gave the best calls over 17 sizes: it reads 35 bytes a ns; it forms 256 x 128 scores and outputs of 128 dims in 7.5
// us (alone 6.0, by which calls where the two kinds nearly balance were up to 15 % slower); a workgroup of either kind begins and ends
// in 6 and 3 us. Own runs have 32 keys at least, and the prefix half the card: `keys` may be a loose bound. (All of the card to the
// prefix first, and then to runs of 128 own keys: 32 sequences of 500 behind 4099 tokens 36 -> 28 us, 16 of 300 behind 16384 39 -> 28,
// 128 of 300 behind 16384 97 -> 83.)
Cut cut_of(int B, int T, int G, int Hkv, int D, int prefix_keys, int keys) {
  Cut c;
  const int rows = B * T * G, tile = tile_keys(D);
  set_form(c, rows, D);
  const int block = 16 * c.rt * c.waves / c.kw;
  c.row_blocks = times(rows, block);
  c.tiles = times(T * G, 16);
  const int tiles = times(prefix_keys, tile), front = Hkv * c.row_blocks, most = 256 / front > 1 ? 256 / front : 1;
  const float read = 4.f * tile * D / 35, form = (float)block * tile * (2 * D + 128) * 6e-4f, a_tile = read > form ? read : form;
  const float a_step = c.waves * (4.f * 32 * D) / 35, a_part = 8.f * Hkv * rows * D / 4900;
  const float late = 35 / 19.f;  // what a step takes longer with all CUs at it
  const int64_t all = (int64_t)B * Hkv * c.tiles;
  float best = INFINITY;
  for (int eighths = 4; eighths <= 8; ++eighths) {
    const int runs = most * eighths / 8 > 1 ? most * eighths / 8 : 1;
    const int span = times(tiles, runs), slots = times(tiles, span);
    const int64_t groups = (int64_t)front * slots;
    const float first = (6000 + span * a_tile) * ((groups + 255) / 256);
    const int64_t left = groups < 256 ? 256 - groups : 0;
    for (int n = 1;; n += (n + 1) / 2) {
      const int run = times(times(keys, n), 32) * 32, own_runs = times(keys, run);
      const int64_t own = (all * own_runs + c.waves - 1) / c.waves;
      const float one = 3000 + run / 32 * a_step;
      // rounds of own workgroups in the CUs left over while the prefix's are at work, and then in all
      const int64_t beside = (int64_t)(first / one) * left;
      float time = first;
      if (own <= left) time = first > one ? first : one;
      else if (own > beside) time = first + (own - beside + 255) / 256 * (3000 + run / 32 * a_step * late);
      time += (slots + own_runs) * a_part;
      if (time < best) {
        best = time;
        c.span = span * tile;
        c.slots = slots;
        c.own_keys = run;
        c.own_runs = own_runs;
      }
      if (run == 32 || own > 4096) break;
    }
    if (runs == most) break;
  }
  return c;
}

struct Plan {
  Cut cut;
  int64_t prefix_groups, groups;  // workgroups
  size_t front, parts, bytes;     // parts of the prefix, and in all
};

Plan plan_of(int B, int T, int Hq, int Hkv, int D, int prefix_keys, int keys) {
  Plan p;
  const int G = Hq / Hkv;
  p.cut = cut_of(B, T, G, Hkv, D, prefix_keys, keys);
  p.prefix_groups = (int64_t)Hkv * p.cut.row_blocks * p.cut.slots;
  p.groups = p.prefix_groups + ((int64_t)B * Hkv * p.cut.tiles * p.cut.own_runs + p.cut.waves - 1) / p.cut.waves;
  p.front = (size_t)B * Hkv * p.cut.slots * T * G;
  p.parts = p.front + (size_t)B * Hkv * p.cut.own_runs * T * G;
  p.bytes = p.parts * (D + 2) * sizeof(float);
  return p;
}

template <int D, int RT, int KW, int NW>
int launch_parts(const Pages& pg, const Prefix& px, const Rows& x, int keys, const Plan& p, hipStream_t s) {
  constexpr int bytes = prefix_lds<D, RT, KW, NW>();
  static_assert(bytes <= 160 * 1024, "a CU's LDS");
  static_assert(bytes >= NW * 16 * D * 4, "a wave's area of its own");
  if (bytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(shared_parts_kernel<D, RT, KW, NW>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return skinny_set_error(SKINNY_ELAUNCH, "paged_attention_shared: %d bytes of LDS: %s", bytes, hipGetErrorString(e));
  }
  hipLaunchKernelGGL((shared_parts_kernel<D, RT, KW, NW>), dim3((uint32_t)p.groups), dim3(64 * NW), bytes, s, pg, px, x,
                     p.cut.row_blocks, p.cut.span, (int)p.prefix_groups, p.cut.tiles, p.cut.own_runs, p.cut.own_keys, keys,
                     x.part_o + p.front * D, x.part_ml + p.front * 2);
  return skinny_check_launch("paged_attention_shared parts");
}

template <int D>
int launch_shared(const Pages& pg, const Prefix& px, const uint16_t* q, int B, int T, int Hq, int Hkv, int keys, float scale,
                  const Plan& p, float* ws, const Out& o, hipStream_t s) {
  float* ml = ws + p.parts * D;
  const Cut& c = p.cut;
  const Rows x{q, B, T, Hq / Hkv, Hq, Hkv, scale, ws, ml};
  auto parts = [&](auto rt, auto kw, auto nw) {
    return launch_parts<D, decltype(rt)::value, decltype(kw)::value, decltype(nw)::value>(pg, px, x, keys, p, s);
  };
  using one = std::integral_constant<int, 1>;
  using two = std::integral_constant<int, 2>;
  using four = std::integral_constant<int, 4>;
  using eight = std::integral_constant<int, 8>;
  int rc;
  if constexpr (D == 256) {
    if (c.kw == 1) rc = parts(one{}, one{}, eight{});
    else if (c.waves == 8) rc = parts(one{}, two{}, eight{});
    else rc = parts(one{}, two{}, four{});
  } else {
    if (c.waves == 4) rc = parts(one{}, four{}, four{});
    else if (c.kw == 1) rc = parts(two{}, one{}, eight{});
    else if (c.kw == 2) rc = parts(two{}, two{}, eight{});
    else if (c.rt == 2) rc = parts(two{}, four{}, eight{});
    else rc = parts(one{}, four{}, eight{});
  }
  if (rc) return rc;
  // Four waves a row while the rows are few (32 heads of 4 sequences behind 20000 tokens 36.8 -> 34.8 us a call, of 128 behind
  // 16384 94.2 -> 99.0; eight waves 36.7 and 108).
  const bool split = (int64_t)B * T * Hq <= 1024;
  auto merge = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(split ? Hq : (Hq + 3) / 4, T, B), dim3(256), 0, s, pg, px, T, Hq, Hq / Hkv, Hkv,
                       keys, c.span, c.own_keys, c.own_runs, p.front, ws, ml, o);
  };
  if (split) merge(shared_merge_kernel<D, 4>);
  else merge(shared_merge_kernel<D, 1>);
  return skinny_check_launch("paged_attention_shared merge");
}

}  // namespace

extern "C" size_t skinny_paged_attn_shared_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int prefix_keys, int keys) {
  if (B < 1 || B > 65535 || T < 1 || Hkv < 1 || Hq < Hkv || Hq > 65535 || Hq % Hkv || !head_dim_ok(D) || keys < 1 ||
      prefix_keys < 1 || prefix_keys > (1 << 30) || keys > (1 << 30) || (int64_t)T * (Hq / Hkv) > kPMaxRows)
    return 0;
  return plan_of(B, T, Hq, Hkv, D, prefix_keys, keys).bytes;
}

extern "C" int skinny_paged_attention_shared_bf16(const uint16_t* q, int B, int T, int Hq, const skinny_paged_kv* kv,
                                                  const int32_t* prefix, const int32_t* prefix_pages, int max_prefix_pages,
                                                  int prefix_keys, int keys, float scale, const uint16_t* gate, int64_t ld_gate,
                                                  int gate_stride, void* workspace, size_t workspace_bytes, uint16_t* out,
                                                  void* stream) {
  Pages pg;
  const char* what = "paged_attention_shared";
  if (const int rc = check_pages(kv, B, T, Hq, pg, what)) return rc;
  const int D = kv->head_dim, Hkv = kv->n_kv;
  SKINNY_CHECK_ARG(q && out && prefix && prefix_pages, "%s: null pointer", what);
  SKINNY_CHECK_ARG((int64_t)T * (Hq / Hkv) <= kPMaxRows, "%s: %lld query rows per kv head, at most %d", what,
                   (long long)T * (Hq / Hkv), kPMaxRows);
  SKINNY_CHECK_ARG(keys >= 1 && keys <= kv->max_pages * kv->page, "%s: keys=%d, the pages hold %d", what, keys,
                   kv->max_pages * kv->page);
  SKINNY_CHECK_ARG(max_prefix_pages >= 1 && (int64_t)max_prefix_pages * kv->page <= (1 << 30) && prefix_keys >= 1 &&
                       prefix_keys <= max_prefix_pages * kv->page,
                   "%s: prefix_keys=%d, %d pages of a prefix", what, prefix_keys, max_prefix_pages);
  SKINNY_CHECK_ARG(!gate || (gate_stride >= 0 && ld_gate >= 0), "%s: gate strides %lld, %d", what, (long long)ld_gate,
                   gate_stride);
  SKINNY_CHECK_ARG(skinny_aligned(q, 16) && skinny_aligned(out, 16) && skinny_aligned(gate, 2) && skinny_aligned(workspace, 16) &&
                       skinny_aligned(prefix, 4) && skinny_aligned(prefix_pages, 4),
                   "%s: misaligned buffer", what);
  SKINNY_CHECK_ARG(scale > 0.f && scale <= 1e38f, "%s: scale=%g must be positive", what, (double)scale);
  const Plan p = plan_of(B, T, Hq, Hkv, D, prefix_keys, keys);
  SKINNY_CHECK_ARG(p.groups <= 0x7fffffff / 8, "%s: keys=%d, prefix_keys=%d of B=%d sequences", what, keys, prefix_keys, B);
  SKINNY_CHECK_ARG(workspace && workspace_bytes >= p.bytes, "%s: workspace of %zu bytes, needs %zu", what,
                   workspace ? workspace_bytes : (size_t)0, p.bytes);
  const Prefix px{prefix, prefix_pages, max_prefix_pages, prefix_keys};
  const Out o{out, gate, ld_gate, gate_stride};
  float* ws = static_cast<float*>(workspace);
  const hipStream_t s = (hipStream_t)stream;
  if (D == 64) return launch_shared<64>(pg, px, q, B, T, Hq, Hkv, keys, scale, p, ws, o, s);
  if (D == 128) return launch_shared<128>(pg, px, q, B, T, Hq, Hkv, keys, scale, p, ws, o, s);
  return launch_shared<256>(pg, px, q, B, T, Hq, Hkv, keys, scale, p, ws, o, s);
}
