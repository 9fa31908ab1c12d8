// Selective state space scan: per head a state h [head_dim][d_state] that decays by exp(d A), takes in (d x) B^T and answers y = h C + D x.
#include "ssm.h"

namespace mb {
namespace ssm {

// exp and the step sizes are the library's fp32 functions: a decay error of one step is taken to the power of the sequence's length
__device__ __forceinline__ float step_size(const mb_selective_scan_args& a, long long at, int head) {
  float d = a.dt_dtype == MB_F32 ? ((const float*)a.d_dt)[at] : a.dt_dtype == MB_F16 ? to_f32(((const f16*)a.d_dt)[at]) : to_f32(((const bf16*)a.d_dt)[at]);
  if (a.d_dt_bias) d += a.d_dt_bias[head];
  if (a.dt_softplus) d = softplus(d);
  return d < a.dt_min ? a.dt_min : d > a.dt_max ? a.dt_max : d;  // NaN stays NaN
}

// Four state columns n .. n+3 of a row; columns from `left` on do not exist and stay zero.  VEC: rows of whole, 16-byte aligned quads.
template <bool VEC> __device__ __forceinline__ f32x4 load_quad(const float* p, int left) {
  if (VEC) return left > 0 ? *(const f32x4*)p : f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) v[i] = p[i];
  return v;
}
template <bool VEC> __device__ __forceinline__ void store_quad(float* p, f32x4 v, int left) {
  if (VEC) {
    if (left > 0) *(f32x4*)p = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) p[i] = v[i];
}
template <typename T> __device__ __forceinline__ f32x4 load_quad_of(const T* p, int left) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) v[i] = to_f32(p[i]);
  return v;
}
template <int LANES> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// One row per item.  LANES lanes hold a state row (4 columns each), 256 / LANES rows at a time; a workgroup takes `pb` rows of one head.
template <typename T, int LANES, bool VEC>
__global__ __launch_bounds__(256) void selective_scan_step_kernel(const mb_selective_scan_args a, int pb) {
  constexpr int ROWS = 256 / LANES;
  const int splits = (a.head_dim + pb - 1) / pb;
  const unsigned item_head = blockIdx.x / splits;
  const int p0 = (int)(blockIdx.x - item_head * splits) * pb;
  const int b = (int)(item_head / a.heads), head = (int)(item_head - (unsigned)b * a.heads);
  const int slot = slot_of(a.d_slots, b, a.n_slots);
  if (slot < 0) return;
  const int n = (int)(threadIdx.x % LANES) * 4, left = a.d_state_dim - n;
  const int group = head / (a.heads / a.groups);
  const float d = step_size(a, b * a.dt_rstride + head, head);
  const float decay = expf(d * a.d_a[head]), skip = a.d_d ? a.d_d[head] : 0.f;
  const f32x4 bv = load_quad_of((const T*)a.d_b + b * a.b_rstride + (long long)group * a.d_state_dim + n, left);
  const f32x4 cv = load_quad_of((const T*)a.d_c + b * a.c_rstride + (long long)group * a.d_state_dim + n, left);
  const T* x = (const T*)a.d_x + b * a.x_rstride + (long long)head * a.head_dim;
  T* y = (T*)a.d_y + b * a.y_rstride + (long long)head * a.head_dim;
  float* h = a.d_state + slot * a.state_stride + (long long)head * a.head_dim * a.d_state_dim + n;
  const int p1 = min(a.head_dim, p0 + pb);
#pragma unroll 4
  for (int p = p0 + (int)threadIdx.x / LANES; p < p1; p += ROWS) {
    f32x4 v = load_quad<VEC>(h + (long long)p * a.d_state_dim, left);
    const float xv = to_f32(x[p]), dx = d * xv;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = fmaf(v[i], decay, dx * bv[i]);
      s = fmaf(v[i], cv[i], s);
    }
    store_quad<VEC>(h + (long long)p * a.d_state_dim, v, left);
    s = lanes_sum<LANES>(s);
    if (n == 0) y[p] = from_f32<T>(fmaf(skip, xv, s));
  }
}

// Row after row: one workgroup per item and head, the head's state in registers (LANES lanes per state row as above).
template <typename T, int LANES, bool VEC>
__global__ __launch_bounds__(256) void selective_scan_rows_kernel(const mb_selective_scan_args a) {
  constexpr int ROWS = 256 / LANES, PASSES = 128 / ROWS > 0 ? 128 / ROWS : 1;
  const int b = (int)(blockIdx.x / a.heads), head = (int)(blockIdx.x - (unsigned)b * a.heads);
  int slot = -1;
  if (a.d_state) {
    slot = slot_of(a.d_slots, b, a.n_slots);
    if (slot < 0) return;
  }
  long long row = 0;
  int len = a.t;
  if (a.d_cu_seqlens) {
    const int s = min(max(a.d_cu_seqlens[b], 0), a.t);
    row = s;
    len = min(max(a.d_cu_seqlens[b + 1], s), a.t) - s;
  } else if (a.d_valid) {
    len = min(max(a.d_valid[b], 0), a.t);
  }
  const long long pad = a.d_cu_seqlens ? 0 : b;
  const int n = (int)(threadIdx.x % LANES) * 4, left = a.d_state_dim - n, p0 = (int)threadIdx.x / LANES;
  const int group = head / (a.heads / a.groups);
  const T* x = (const T*)a.d_x + pad * a.x_bstride + row * a.x_rstride + (long long)head * a.head_dim;
  T* y = (T*)a.d_y + pad * a.y_bstride + row * a.y_rstride + (long long)head * a.head_dim;
  const T* bm = (const T*)a.d_b + pad * a.b_bstride + row * a.b_rstride + (long long)group * a.d_state_dim + n;
  const T* cm = (const T*)a.d_c + pad * a.c_bstride + row * a.c_rstride + (long long)group * a.d_state_dim + n;
  const long long dt = pad * a.dt_bstride + row * a.dt_rstride + head;
  float* st = a.d_state ? a.d_state + slot * a.state_stride + (long long)head * a.head_dim * a.d_state_dim + n : nullptr;
  const bool keep = st && (!a.d_has_state || a.d_has_state[b]);
  const float A = a.d_a[head], skip = a.d_d ? a.d_d[head] : 0.f;
  f32x4 h[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int p = p0 + i * ROWS;
    h[i] = keep && p < a.head_dim ? load_quad<VEC>(st + (long long)p * a.d_state_dim, left) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int t = 0; t < len; ++t) {
    const float d = step_size(a, dt + t * a.dt_rstride, head), decay = expf(d * A);
    const f32x4 bv = load_quad_of(bm + t * a.b_rstride, left), cv = load_quad_of(cm + t * a.c_rstride, left);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int p = p0 + i * ROWS;
      const float xv = p < a.head_dim ? to_f32(x[t * a.x_rstride + p]) : 0.f, dx = d * xv;
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        h[i][k] = fmaf(h[i][k], decay, dx * bv[k]);
        s = fmaf(h[i][k], cv[k], s);
      }
      s = lanes_sum<LANES>(s);
      if (n == 0 && p < a.head_dim) y[t * a.y_rstride + p] = from_f32<T>(fmaf(skip, xv, s));
    }
  }
  if (st)
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int p = p0 + i * ROWS;
      if (p < a.head_dim) store_quad<VEC>(st + (long long)p * a.d_state_dim, h[i], left);
    }
}

template <typename T, int LANES, bool VEC> int launch_scan(const mb_selective_scan_args& a, bool step, hipStream_t s) {
  if (step) {
    constexpr int ROWS = 256 / LANES;
    int pb = (a.head_dim + ROWS - 1) / ROWS * ROWS;
    // few requests: a head's rows are dealt to more workgroups, down to one pass each, until two fit every CU
    while (pb > ROWS && (long long)a.batch * a.heads * ((a.head_dim + pb - 1) / pb) < 512) pb = (pb / ROWS + 1) / 2 * ROWS;
    const long long grid = (long long)a.batch * a.heads * ((a.head_dim + pb - 1) / pb);
    MB_REQUIRE(grid < (1ll << 31), "selective_scan_step: %d items of %d heads are too many for one launch", a.batch, a.heads);
    hipLaunchKernelGGL((selective_scan_step_kernel<T, LANES, VEC>), dim3((unsigned)grid), dim3(256), 0, s, a, pb);
  } else {
    MB_REQUIRE((long long)a.batch * a.heads < (1ll << 31), "selective_scan: %d items of %d heads are too many for one launch", a.batch, a.heads);
    hipLaunchKernelGGL((selective_scan_rows_kernel<T, LANES, VEC>), dim3((unsigned)(a.batch * a.heads)), dim3(256), 0, s, a);
  }
  MB_HIP(hipGetLastError());
  return MB_OK;
}

template <typename T, bool VEC> int scan_by_lanes(const mb_selective_scan_args& a, bool step, hipStream_t s) {
  if (a.d_state_dim <= 16) return launch_scan<T, 4, VEC>(a, step, s);
  if (a.d_state_dim <= 32) return launch_scan<T, 8, VEC>(a, step, s);
  if (a.d_state_dim <= 64) return launch_scan<T, 16, VEC>(a, step, s);
  if (a.d_state_dim <= 128) return launch_scan<T, 32, VEC>(a, step, s);
  return launch_scan<T, 64, VEC>(a, step, s);
}

template <typename T> int scan_by_width(const mb_selective_scan_args& a, bool step, hipStream_t s) {
  const bool vec = a.d_state_dim % 4 == 0 && (!a.d_state || (aligned(a.d_state, 16) && a.state_stride % 4 == 0));
  return vec ? scan_by_lanes<T, true>(a, step, s) : scan_by_lanes<T, false>(a, step, s);
}

static int check_scan(const char* name, const mb_selective_scan_args* a, bool step) {
  MB_REQUIRE(a, "%s: null arguments", name);
  MB_REQUIRE(a->dtype == MB_F32 || a->dtype == MB_F16 || a->dtype == MB_BF16, "%s: dtype %d is none of MB_F32, MB_F16, MB_BF16", name, a->dtype);
  MB_REQUIRE(a->dt_dtype == a->dtype || a->dt_dtype == MB_F32, "%s: dt_dtype %d is neither dtype nor MB_F32", name, a->dt_dtype);
  MB_REQUIRE(a->batch >= 0 && a->heads >= 0 && (step || a->t >= 0), "%s: negative shape", name);
  MB_REQUIRE(a->head_dim >= 1 && a->head_dim <= 128, "%s: head_dim %d is outside 1..128", name, a->head_dim);
  MB_REQUIRE(a->d_state_dim >= 1 && a->d_state_dim <= 256, "%s: d_state %d is outside 1..256", name, a->d_state_dim);
  MB_REQUIRE(a->groups >= 1 && a->heads % a->groups == 0, "%s: %d heads in %d groups", name, a->heads, a->groups);
  MB_REQUIRE(a->dt_min <= a->dt_max, "%s: dt_min %g, dt_max %g", name, a->dt_min, a->dt_max);  // refuses NaN as well
  if (a->batch == 0 || a->heads == 0) return MB_OK;
  MB_REQUIRE(a->d_a, "%s: no A", name);
  MB_REQUIRE((a->d_x && a->d_y && a->d_dt && a->d_b && a->d_c) || (!step && a->t == 0), "%s: null x, y, dt, B or C", name);
  MB_REQUIRE(!step || a->d_state, "%s: a step needs a state pool", name);
  if (a->d_state) {
    MB_REQUIRE(a->n_slots >= 0 && a->state_stride >= 0, "%s: negative state pool", name);
    MB_REQUIRE(a->d_slots || a->batch <= a->n_slots, "%s: %d items without slot numbers, but %d slots", name, a->batch, a->n_slots);
  } else {
    MB_REQUIRE(!a->d_slots && !a->d_has_state, "%s: slots or has_state without a state pool", name);
  }
  MB_REQUIRE(!a->d_cu_seqlens || !a->d_valid, "%s: packed and padded rows at once", name);
  MB_REQUIRE(!a->d_cu_seqlens || (long long)a->t + a->batch < (1ll << 31), "%s: %d rows of %d items are too many", name, a->t, a->batch);
  return 1;
}

static int run_scan(const char* name, const mb_selective_scan_args* a, bool step, mb_stream_t stream) {
  const int go = check_scan(name, a, step);
  if (go <= 0) return go;
  if (a->dtype == MB_F32) return scan_by_width<float>(*a, step, (hipStream_t)stream);
  if (a->dtype == MB_F16) return scan_by_width<f16>(*a, step, (hipStream_t)stream);
  return scan_by_width<bf16>(*a, step, (hipStream_t)stream);
}

}  // namespace ssm
}  // namespace mb

extern "C" size_t mb_selective_scan_workspace_bytes(const mb_selective_scan_args* a) { return 0; }
extern "C" int mb_selective_scan(const mb_selective_scan_args* a, void* d_workspace, size_t workspace_bytes, mb_stream_t stream) {
  return mb::ssm::run_scan("selective_scan", a, false, stream);
}
extern "C" int mb_selective_scan_step(const mb_selective_scan_args* a, mb_stream_t stream) {
  return mb::ssm::run_scan("selective_scan_step", a, true, stream);
}
