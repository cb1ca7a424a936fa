// What the kernels over a cache in pages share (paged.hip, paged_shared.hip): the cache as they see it, the parts of a
// softmax and how they are joined, and the checks of the cache's description.
#pragma once

#include "common.h"

namespace paged {

constexpr float kPLog2e = 1.4426950408889634f;
constexpr int kPMaxRows = 64;  // query rows per kv head: T x (Hq / Hkv)

// Memory that a kernel only reads, for uniform addresses: loaded into scalar registers.
typedef const __attribute__((address_space(4))) int32_t* words_t;
__device__ __forceinline__ words_t words(const int32_t* p) { return (words_t)(uintptr_t)p; }

struct Pages {
  const int32_t* lengths;
  const int32_t* counts;  // null: T each
  const int32_t* table;   // [B][>= max_pages], row stride ld
  uint16_t* k;
  uint16_t* vt;
  uint32_t k_stride, vt_stride;  // elements from page to page
  int ld, max_pages, n_pages, log2p;
};

// A sequence's cached length and new tokens. `ok` is false where they cannot be: a negative length, a count
// outside [0, T], or more tokens than `room` slots.
struct Sequence {
  int len, count;
  bool ok;
};
__device__ __forceinline__ Sequence sequence_of(const Pages& pg, int b, int T, int room) {
  const int len = words(pg.lengths)[b], count = pg.counts ? words(pg.counts)[b] : T;
  return {len, count, len >= 0 && count >= 0 && count <= T && count <= room && len <= room - count};
}

constexpr uint16_t kNanBits = 0x7fc0;

typedef __attribute__((ext_vector_type(2))) float f32x2_t;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
__device__ __forceinline__ uint32_t two_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
}

// The first n (0 to 8) of eight consecutive keys' values, the others zero.
__device__ __forceinline__ u32x4_t first_keys(u32x4_t v, int n) {
#pragma unroll
  for (int w = 0; w < 4; ++w) v[w] &= n >= 2 * w + 2 ? ~0u : n == 2 * w + 1 ? 0xffffu : 0u;
  return v;
}

struct Out {
  uint16_t* out;
  const uint16_t* gate;  // null: none
  int64_t ldg;           // elements from row to row
  int gs;                // and from head to head
};

// One output value, divided by the sum of its weights, gated, rounded. Sums that are not finite end here as one NaN: a value
// that is not finite leaves an infinity or a NaN, by the sign of its weight's second term, which the joins keep (times a
// factor that is no 0 or, of 0, as NaN). A compare and a select per value; no block pays for it.
__device__ __forceinline__ uint16_t finished(float o, float inv, bool gated, uint32_t gate) {
  o *= inv;
  const bool finite = fabsf(o) < INFINITY;
  if (gated) o *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(bf16_bits_to_f32(gate) * -kPLog2e));
  return finite ? f32_to_bf16_bits(o) : kNanBits;
}

// Part (m, l, o) of a row joined to the parts before it: their factor and its own.
struct Join {
  float before, part;
};
__device__ __forceinline__ Join join(float& m, float& l, float pm, float pl) {
  const float mm = fmaxf(m, pm), ref = mm == -INFINITY ? 0.f : mm;
  const Join j{__builtin_amdgcn_exp2f(m - ref), __builtin_amdgcn_exp2f(pm - ref)};
  m = mm;
  l = fmaf(pl, j.part, l * j.before);
  return j;
}

// The larger of, and the sum over, the four quads' values of a column, in every lane.
__device__ __forceinline__ float quads_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quads_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

inline bool head_dim_ok(int D) { return D == 64 || D == 128 || D == 256; }

// What both entry points ask of the cache; sets `pg`.
inline int check_pages(const skinny_paged_kv* kv, int B, int T, int Hq, Pages& pg, const char* what) {
  SKINNY_CHECK_ARG(kv && kv->lengths && kv->pages && kv->k_pages && kv->vt_pages, "%s: null pointer", what);
  SKINNY_CHECK_ARG(head_dim_ok(kv->head_dim), "%s: head dim %d unsupported (64, 128 or 256)", what, kv->head_dim);
  SKINNY_CHECK_ARG(kv->n_kv >= 1 && kv->n_kv <= 32767 && Hq >= kv->n_kv && Hq <= 65535 && Hq % kv->n_kv == 0,
                   "%s: Hq=%d must be a multiple of Hkv=%d", what, Hq, kv->n_kv);
  SKINNY_CHECK_ARG(B >= 1 && B <= 65535 && T >= 1 && T <= 65535, "%s: B=%d sequences of T=%d tokens (1 to 65535 each)",
                   what, B, T);
  const int P = kv->page;
  SKINNY_CHECK_ARG(P >= 16 && P <= 256 && (P & (P - 1)) == 0, "%s: page=%d slots (a power of two, 16 to 256)", what, P);
  SKINNY_CHECK_ARG(kv->n_pages >= 1 && kv->max_pages >= 1 && kv->ld_pages >= kv->max_pages &&
                       (int64_t)kv->max_pages * P <= (1 << 30),
                   "%s: n_pages=%d, max_pages=%d, ld_pages=%d", what, kv->n_pages, kv->max_pages, kv->ld_pages);
  const int64_t need = (int64_t)kv->n_kv * P * kv->head_dim;
  SKINNY_CHECK_ARG(kv->k_stride >= need && kv->vt_stride >= need && kv->k_stride % 8 == 0 && kv->vt_stride % 8 == 0 &&
                       kv->k_stride <= INT32_MAX && kv->vt_stride <= INT32_MAX,
                   "%s: page strides %lld, %lld (multiples of 8 below 2^31, at least Hkv*P*D=%lld)", what,
                   (long long)kv->k_stride, (long long)kv->vt_stride, (long long)need);
  SKINNY_CHECK_ARG(skinny_aligned(kv->k_pages, 16) && skinny_aligned(kv->vt_pages, 16) && skinny_aligned(kv->lengths, 4) &&
                       skinny_aligned(kv->counts, 4) && skinny_aligned(kv->pages, 4),
                   "%s: misaligned cache", what);
  pg = Pages{kv->lengths, kv->counts, kv->pages, kv->k_pages, kv->vt_pages, (uint32_t)kv->k_stride, (uint32_t)kv->vt_stride,
             kv->ld_pages, kv->max_pages, kv->n_pages, __builtin_ctz(P)};
  return SKINNY_OK;
}

}  // namespace paged
