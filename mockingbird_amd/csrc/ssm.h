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

// softplus without overflow: max(v, 0) + log(1 + exp(-|v|)); NaN stays NaN
__device__ __forceinline__ float softplus(float v) { return (v > 0.f ? v : 0.f) + log1pf(expf(-fabsf(v))); }

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
// Tiles never cross an item.  Packed: item b owns the tile numbers from cu[b] / R + b on.  With s = a R + u and len = c R + v the next
// item starts at least c + 1 >= ceil(len / R) numbers later, so the ranges are disjoint and every item has a tile 0, also an empty one;
// t / R + batch numbers cover all.  No prefix sum over the items, and the host needs no lengths.
__host__ __device__ inline long long tiles_of(const Rows& r, int R) {
  return r.cu ? (long long)r.t / R + r.batch : (long long)r.batch * (r.t > R ? (r.t + R - 1) / R : 1);
}
__device__ __forceinline__ Item item_of(const Rows& r, unsigned tile, int R) {
  Item it;
  if (r.cu) {
    int lo = 0, hi = r.batch - 1;
    while (lo < hi) {  // the last item whose first tile is <= tile
      const int mid = (lo + hi + 1) >> 1;
      const int s = min(max(r.cu[mid], 0), r.t);
      if (s / R + mid <= (int)tile) lo = mid; else hi = mid - 1;
    }
    const int s = min(max(r.cu[lo], 0), r.t), e = min(max(r.cu[lo + 1], s), r.t);
    it.b = lo; it.len = e - s; it.row = s; it.part = (int)tile - (s / R + lo);
  } else {
    const unsigned per = r.t > R ? (unsigned)(r.t + R - 1) / R : 1u;
    it.b = (int)(tile / per);
    it.part = (int)(tile - (unsigned)it.b * per);
    it.len = r.valid ? min(max(r.valid[it.b], 0), r.t) : r.t;
    it.row = 0;
  }
  return it;
}

// Slot of item b, or -1: outside the pool, or named by an earlier item as well (two updates of one state would race; the first wins).
// Wave-uniform; every lane of the wave calls it.
__device__ __forceinline__ int slot_of(const int* slots, int b, int n_slots) {
  if (!slots) return b;
  const int s = slots[b];
  if (s < 0 || s >= n_slots) return -1;
  bool twice = false;
  for (int i = (int)(threadIdx.x & 63); i < b; i += 64) twice |= slots[i] == s;
  return __any(twice) ? -1 : s;
}

__host__ __device__ static inline bool aligned(const void* p, size_t n) { return ((size_t)p & (n - 1)) == 0; }

}  // namespace ssm
}  // namespace mb
