// Shared by the state-space block kernels (ssm_conv.hip, ssm_scan.hip, ssm_norm.hip): element types, the map from workgroups to the
// rows of an item, state slots.
#pragma once
#include <type_traits>
#include "common.h"

namespace mb {
namespace ssm {

typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }  // one rounding to nearest even

// N elements as one access.  Rows start at any element (odd widths, slices), so the accesses ask for the element's alignment only: global
// memory takes a 16-byte access at any address, at the price of the extra cache line it may touch.
template <typename T, int N> struct Vec { T v[N]; };
template <typename T, int N> __device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
  typedef T vt __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  return __builtin_bit_cast(Vec<T, N>, *(const vt*)p);
}
template <typename T, int N> __device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& v) {
  typedef T vt __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  *(vt*)p = __builtin_bit_cast(vt, v);
}
// The first n of N elements (the rest are zero / left alone): the end of a row whose width N does not divide.
template <typename T, int N> __device__ __forceinline__ Vec<T, N> load_some(const T* p, int n) {
  Vec<T, N> v;
  if (n >= N) return load_vec<T, N>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v.v[i] = (T)0.f;
    if (i < n) v.v[i] = p[i];
  }
  return v;
}
template <typename T, int N> __device__ __forceinline__ void store_some(T* p, const Vec<T, N>& v, int n) {
  if (n >= N) return store_vec<T, N>(p, v);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) p[i] = v.v[i];
}

// exp and 1 / (1 + exp(-v)).  fp32 results go through the library's expf and a full division; a 16-bit result is rounded to 2^-9 or
// 2^-12 relative, so v_exp_f32 on a rounded argument (relative error |v| 2^-24, 1e-5 where the sigmoid is still above 2^-126) is enough.
template <bool FAST> __device__ __forceinline__ float sigmoid(float v) {
  if (FAST) return __builtin_amdgcn_rcpf(1.f + __expf(-v));
  return 1.f / (1.f + expf(-v));
}

// exp to about an ulp: the product with log2(e) is taken in two parts, the second as a first-order factor.  (Not for |v| beyond 2^7 or so.)
__device__ __forceinline__ float exp_of(float v) {
  const float p = v * 1.44269502f, rest = fmaf(v, 1.92596299e-8f, fmaf(v, 1.44269502f, -p));
  const float e = __builtin_amdgcn_exp2f(p);
  return fmaf(e, rest * 0.693147182f, e);
}
// softplus without overflow: max(v, 0) + log(1 + e), e = exp(-|v|).  The rounding of 1 + e is taken out again by e / ((1 + e) - 1): a few
// units in the last place at any v.  NaN stays NaN.
__device__ __forceinline__ float softplus(float v) {
  const float e = exp_of(-(fabsf(v) > 120.f ? 120.f : fabsf(v))), one = 1.f + e, less = one - 1.f;
  const float log1p = less == 0.f ? e : __builtin_amdgcn_logf(one) * 0.693147182f * (e * __builtin_amdgcn_rcpf(less));
  return (v > 0.f ? v : 0.f) + log1p;
}

// Rows of one call: packed (cu) or padded (valid).  Everything read from the device is clamped to 0..t, so that no list of row numbers
// can lead outside the tensors.
struct Rows {
  const int* cu;
  const int* valid;
  int batch, t;
};
struct Item {
  int b;         // item
  int len;       // its rows
  long long row; // its first row on the packed row axis (0 when padded)
  int part;      // which tile of it
};
// Tiles of R rows never cross an item; an item without rows has one (its state is still to be written).  Without lengths on the device every
// item has the same number of them.  Otherwise they are numbered without gaps -- a gap would be an idle workgroup, and idle ones that
// alternate with busy ones in dispatch order land on the same shader engines -- from the lengths themselves: 64 items are summed up at a
// time by the lanes of each wave.  The host needs no lengths, only the bound tiles_of (the numbers behind the last tile are idle).
__host__ __device__ inline long long tiles_of(const Rows& r, int R) {
  return r.cu ? (long long)r.t / R + r.batch : (long long)r.batch * (r.t > R ? (r.t + R - 1) / R : 1);
}
__device__ __forceinline__ int rows_of(const Rows& r, int b, int& first) {
  if (r.cu) {
    first = min(max(r.cu[b], 0), r.t);
    return min(max(r.cu[b + 1], first), r.t) - first;
  }
  first = 0;
  return r.valid ? min(max(r.valid[b], 0), r.t) : r.t;
}
__device__ __forceinline__ int lanes_prefix(int v) {  // inclusive, over the wave
  const int lane = (int)threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int up = __shfl_up(v, o, 64);
    v += lane >= o ? up : 0;
  }
  return v;
}
// part < 0: no such tile.  Every lane of the wave calls it with the same tile.  less = 1: all but the last tile of each item are numbered.
__device__ __forceinline__ Item item_of(const Rows& r, unsigned tile, int R, int less = 0) {
  Item it = {0, 0, 0, -1};
  if (!r.cu && !r.valid) {
    const unsigned per = (r.t > R ? (unsigned)(r.t + R - 1) / R : 1u) - less;
    it.b = (int)(tile / per);
    it.part = (int)(tile - (unsigned)it.b * per);
    it.len = r.t;
    return it;
  }
  int base = 0;
  for (int i0 = 0; i0 < r.batch; i0 += 64) {
    const int i = i0 + ((int)threadIdx.x & 63);
    int first = 0, len = 0, parts = 0;
    if (i < r.batch) {
      len = rows_of(r, i, first);
      parts = max(1, (len + R - 1) / R) - less;
    }
    const int end = base + lanes_prefix(parts);
    const unsigned long long behind = __ballot(end > (int)tile);
    if (behind) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll((long long)behind) - 1);  // scalars from here on
      it.b = i0 + l;
      it.len = __builtin_amdgcn_readlane(len, l);
      it.row = __builtin_amdgcn_readlane(first, l);
      it.part = (int)tile - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(parts, l));
      return it;
    }
    base = __builtin_amdgcn_readlane(end, 63);
  }
  return it;
}
// The items of more than one tile, for calls whose tiles need a place in memory: together they have at most this many tiles in front of
// their last ones, whatever the number of items.  (t > R)
__host__ __device__ inline long long fronts_of(const Rows& r, int R) {
  return r.cu ? (long long)r.t / R : (long long)r.batch * ((r.t + R - 1) / R - 1);
}
// The j-th of them (b < 0: there are not so many), its tiles, and how many tiles in front of last ones the items before it have.  Every lane
// of the wave calls it with the same j.
struct Long {
  int b, parts, fronts;
};
__device__ __forceinline__ Long long_item(const Rows& r, int j, int R) {
  if (!r.cu && !r.valid) {
    const int parts = (r.t + R - 1) / R;
    return {j, parts, j * (parts - 1)};
  }
  int items = 0, fronts = 0;
  for (int i0 = 0; i0 < r.batch; i0 += 64) {
    const int i = i0 + ((int)threadIdx.x & 63);
    int first, parts = 1;
    if (i < r.batch) parts = max(1, (rows_of(r, i, first) + R - 1) / R);
    const int upto = items + lanes_prefix(parts > 1), before = fronts + lanes_prefix(parts - 1) - (parts - 1);
    const unsigned long long behind = __ballot(upto > j);
    if (behind) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll((long long)behind) - 1);
      return {i0 + l, __builtin_amdgcn_readlane(parts, l), __builtin_amdgcn_readlane(before, l)};
    }
    items = __builtin_amdgcn_readlane(upto, 63);
    // (lists of overlapping rows could claim any number of tiles: 64 items have at most 2^30, and the sum stops there)
    fronts = min(__builtin_amdgcn_readlane(before + (parts - 1), 63), (1 << 30) - 1);
  }
  return {-1, 0, 0};
}

// Slot of item b, or -1: outside the pool, or named by an earlier item as well (two updates of one state would race; the first wins).
// Wave-uniform; every lane of the wave calls it.
__device__ __forceinline__ int slot_of(const int* slots, int b, int n_slots) {
  if (!slots) return b;
  const int s = __builtin_amdgcn_readfirstlane(slots[b]);
  if (s < 0 || s >= n_slots) return -1;
  bool twice = false;
  for (int i = (int)(threadIdx.x & 63); i < b; i += 64) twice |= slots[i] == s;
  return __any(twice) ? -1 : s;
}

// A tensor of a call, for the check of what shares memory: a run of `bytes`, repeated along up to three axes (innermost first).
struct Span {
  const char* name;
  const void* p;
  long long bytes, n[3], stride[3];
};
static inline Span span_of(const char* name, const void* p, size_t elem, long long run, long long n0 = 1, long long s0 = 0, long long n1 = 1, long long s1 = 0) {
  return {name, p, run * (long long)elem, {n0, n1, 1}, {s0 * (long long)elem, s1 * (long long)elem, 0}};
}
// Its address range; empty without a tensor.
static inline void range_of(const Span& s, __int128& lo, __int128& hi) {
  lo = hi = (__int128)(size_t)s.p;
  if (!s.p || s.bytes <= 0) return;
  __int128 down = 0, up = s.bytes;
  for (int i = 0; i < 3; ++i) {
    if (s.n[i] <= 0) return;
    (s.stride[i] < 0 ? down : up) += (__int128)(s.n[i] - 1) * s.stride[i];
  }
  lo += down, hi += up;
}
// Two tensors whose ranges overlap share nothing if both repeat a run at multiples of one step (rows of a wider buffer) and the runs lie in
// different columns of it.
static inline bool other_columns(const Span& a, const Span& b) {
  const Span* const s[2] = {&a, &b};
  __int128 run[2], front[2][3], step = 0;
  int axes[2];
  for (int k = 0; k < 2; ++k) {
    run[k] = s[k]->bytes, axes[k] = 0;
    for (int i = 0; i < 3; ++i) {
      const __int128 n = s[k]->n[i], st = s[k]->stride[i] < 0 ? -(__int128)s[k]->stride[i] : s[k]->stride[i];
      if (n == 1) continue;
      if (!axes[k] && s[k]->stride[i] == run[k]) {
        run[k] *= n;
      } else {
        front[k][axes[k]++] = st;
        if (st && (!step || st < step)) step = st;
      }
    }
  }
  if (!step) return false;
  for (int k = 0; k < 2; ++k)
    for (int i = 0; i < axes[k]; ++i)
      if (front[k][i] % step) return false;
  const __int128 off = (((__int128)(size_t)b.p - (__int128)(size_t)a.p) % step + step) % step;
  return off >= run[0] && off + run[1] <= step;
}
// What a call writes (the first `written` spans) overlaps none of its other tensors; from `same` on a span may be exactly a written one.
static inline int check_apart(const char* fn, const Span* s, int written, int all, int same = 16) {
  __int128 lo[16], hi[16];
  for (int i = 0; i < all; ++i) range_of(s[i], lo[i], hi[i]);
  for (int i = 0; i < written; ++i)
    for (int j = i + 1; j < all; ++j) {
      if (lo[i] >= hi[j] || lo[j] >= hi[i]) continue;
      const bool equal = j >= same && s[i].p == s[j].p && s[i].bytes == s[j].bytes && (s[i].n[0] == 1 || s[i].stride[0] == s[j].stride[0]);
      MB_REQUIRE(equal || other_columns(s[i], s[j]), "%s: %s overlaps %s", fn, s[i].name, s[j].name);
    }
  return MB_OK;
}

__host__ __device__ static inline bool aligned(const void* p, size_t n) { return ((size_t)p & (n - 1)) == 0; }
static inline bool launchable(long long workgroups, int threads) { return workgroups < (1ll << 31) && workgroups * threads < (1ll << 32); }
static inline size_t size_of(int dtype) { return dtype == MB_F32 ? 4 : 2; }

}  // namespace ssm
}  // namespace mb
