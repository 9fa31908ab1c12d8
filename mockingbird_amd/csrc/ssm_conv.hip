// Short causal depthwise convolution over rows of channels, with the last inputs of every item kept as its state.
//   y[t][c] = act(bias[c] + sum_j w[c][j] x[t - K + 1 + j][c])
#include "ssm.h"

namespace mb {
namespace ssm {

// The taps of V channels: one run of V * K floats.
template <int K, int V> __device__ __forceinline__ void load_taps(const float* w, int n, float (&out)[V][K]) {
  if (n >= V) {
    constexpr int Q = V * K / 4;
    Vec<float, 4> q[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) q[i] = load_vec<float, 4>(w + 4 * i);
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < K; ++j) out[i][j] = q[(i * K + j) / 4].v[(i * K + j) % 4];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < K; ++j) out[i][j] = i < n ? w[i * K + j] : 0.f;
  }
}

// A thread takes 4 channels of R rows, cx threads side by side and 256 / cx runs of R rows behind each other.  Memory-bound: each row is
// read once (a run reads K - 1 more) and the window slides through registers; U rows are requested at a time.  8 channels of a 16-bit type
// (16 bytes) need 146 registers for window and taps and run at 2.7 TB/s for want of waves, 4 channels at 5.0 TB/s (16 k rows of 4352
// channels, 4 taps: 108 and 58 us); rows of fp32 are 16 bytes either way.  Runs of 16 to 64 rows differ by 5 %.
constexpr int CONV_V = 4;
template <typename T, int K>
__global__ __launch_bounds__(256) void causal_conv1d_kernel(const mb_causal_conv1d_args a, int cx, int R) {
  constexpr bool FAST = sizeof(T) == 2;
  constexpr int V = CONV_V, U = 4;
  const int ci = threadIdx.x & (cx - 1), rg = threadIdx.x / cx, groups = 256 / cx;
  const int blocks_c = (a.channels + cx * V - 1) / (cx * V);
  const unsigned tile = blockIdx.x / blocks_c;
  const int c = ((int)(blockIdx.x - tile * blocks_c) * cx + ci) * V, n = a.channels - c;
  const Rows rows = {a.d_cu_seqlens, a.d_valid, a.batch, a.t};
  const Item it = item_of(rows, tile, R * groups);
  if (it.part < 0 || it.part >= max(1, (it.len + R * groups - 1) / (R * groups))) return;
  int slot = -1;
  if (a.d_state) {
    slot = slot_of(a.d_slots, it.b, a.n_slots);
    if (slot < 0) return;
  }
  if (n <= 0) return;
  const T* x = (const T*)a.d_x + it.row * a.x_rstride + (a.d_cu_seqlens ? 0 : it.b * a.x_bstride) + c;
  T* y = (T*)a.d_y + it.row * a.y_rstride + (a.d_cu_seqlens ? 0 : it.b * a.y_bstride) + c;
  const int t0 = (it.part * groups + rg) * R, t1 = min(it.len, t0 + R);
  const bool first = it.part == 0 && rg == 0;
  if (!first && t0 >= t1) return;
  Vec<T, V> win[K - 1];  // rows t - K + 1 .. t - 1
  if (first) {
    T* st = a.d_state ? (T*)a.d_state + slot * a.state_stride + c : nullptr;
    const bool keep = st && (!a.d_has_state || a.d_has_state[it.b]);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) win[j] = load_some<T, V>(st + (long long)j * a.channels, keep ? n : 0);
    if (st) {  // only this thread touches these channels of the slot: the old rows are in registers before the new ones are written
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        const int from = it.len + j;  // row of (state ++ x): the last K - 1 of it
        Vec<T, V> v;
        if (from >= K - 1) {
          v = load_some<T, V>(x + (from - (K - 1)) * a.x_rstride, n);
        } else {
#pragma unroll
          for (int k = 0; k < K - 1; ++k)
            if (k == from) v = win[k];
        }
        store_some<T, V>(st + (long long)j * a.channels, v, n);
      }
    }
    if (t0 >= t1) return;
  } else {  // R >= K - 1: these rows are the item's own
#pragma unroll
    for (int j = 0; j < K - 1; ++j) win[j] = load_some<T, V>(x + (t0 - (K - 1) + j) * a.x_rstride, n);
  }
  float w[V][K], line[K - 1 + U][V];
  load_taps<K, V>(a.d_w + (long long)c * K, n, w);
  const Vec<float, V> bias = load_some<float, V>(a.d_bias + c, a.d_bias ? n : 0);
#pragma unroll
  for (int j = 0; j < K - 1; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) line[j][i] = to_f32(win[j].v[i]);
  for (int t = t0; t < t1; t += U) {
    Vec<T, V> cur[U];
#pragma unroll
    for (int u = 0; u < U; ++u) cur[u] = load_some<T, V>(x + min(t + u, t1 - 1) * a.x_rstride, n);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Vec<T, V> out;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        line[K - 1 + u][i] = to_f32(cur[u].v[i]);
        float v = bias.v[i];
#pragma unroll
        for (int j = 0; j < K; ++j) v = fmaf(w[i][j], line[u + j][i], v);
        if (a.act) v *= sigmoid<FAST>(v);
        out.v[i] = from_f32<T>(v);
      }
      if (t + u < t1) store_some<T, V>(y + (t + u) * a.y_rstride, out, n);
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) line[j][i] = line[j + U][i];
  }
}

// One row per item: the same sum with the state as the window; the state moves up by one row in place.
template <typename T, int K>
__global__ __launch_bounds__(64) void causal_conv1d_step_kernel(const mb_causal_conv1d_args a) {
  constexpr bool FAST = sizeof(T) == 2;
  constexpr int V = CONV_V;
  const int per = (a.channels + 64 * V - 1) / (64 * V);
  const int b = (int)(blockIdx.x / per);
  const int c = ((int)(blockIdx.x - (unsigned)b * per) * 64 + (int)threadIdx.x) * V, n = a.channels - c;
  const int slot = slot_of(a.d_slots, b, a.n_slots);
  if (slot < 0 || n <= 0) return;
  const Vec<T, V> cur = load_some<T, V>((const T*)a.d_x + b * a.x_rstride + c, n);
  T* st = (T*)a.d_state + slot * a.state_stride + c;
  Vec<T, V> win[K - 1], out;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) win[j] = load_some<T, V>(st + (long long)j * a.channels, n);
  float w[V][K];
  load_taps<K, V>(a.d_w + (long long)c * K, n, w);
  const Vec<float, V> bias = load_some<float, V>(a.d_bias + c, a.d_bias ? n : 0);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float v = bias.v[i];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) v = fmaf(w[i][j], to_f32(win[j].v[i]), v);
    v = fmaf(w[i][K - 1], to_f32(cur.v[i]), v);
    if (a.act) v *= sigmoid<FAST>(v);
    out.v[i] = from_f32<T>(v);
  }
  store_some<T, V>((T*)a.d_y + b * a.y_rstride + c, out, n);
#pragma unroll
  for (int j = 0; j + 1 < K - 1; ++j) store_some<T, V>(st + (long long)j * a.channels, win[j + 1], n);
  store_some<T, V>(st + (long long)(K - 2) * a.channels, cur, n);
}

static int conv_apart(const char* name, const mb_causal_conv1d_args& a, bool step) {
  const size_t e = size_of(a.dtype);
  const bool padded = !step && !a.d_cu_seqlens;
  const long long rows = step ? a.batch : a.t, items = padded ? a.batch : 1;
  const Span s[] = {span_of("out", a.d_y, e, a.channels, rows, a.y_rstride, items, a.y_bstride),
                    span_of("state", a.d_state, e, (long long)(a.ksize - 1) * a.channels, a.n_slots, a.state_stride),
                    span_of("x", a.d_x, e, a.channels, rows, a.x_rstride, items, a.x_bstride),
                    span_of("weight", a.d_w, 4, (long long)a.channels * a.ksize),
                    span_of("bias", a.d_bias, 4, a.channels),
                    span_of("slots", a.d_slots, 4, a.batch),
                    span_of("has_state", step ? nullptr : a.d_has_state, 1, a.batch),
                    span_of("cu_seqlens", step ? nullptr : a.d_cu_seqlens, 4, a.batch + 1ll),
                    span_of("lengths", step ? nullptr : a.d_valid, 4, a.batch)};
  return check_apart(name, s, 2, sizeof(s) / sizeof(*s));
}

template <typename T, int K> int launch_conv(const mb_causal_conv1d_args& a, bool step, hipStream_t s) {
  if (step) {
    const long long grid = (long long)a.batch * cdiv(a.channels, 64 * CONV_V);
    MB_REQUIRE(launchable(grid, 64), "causal_conv1d_step: %d items of %d channels are too many for one launch", a.batch, a.channels);
    if (const int rc = conv_apart("causal_conv1d_step", a, true)) return rc;
    hipLaunchKernelGGL((causal_conv1d_step_kernel<T, K>), dim3((unsigned)grid), dim3(64), 0, s, a);
  } else {
    const int nv = cdiv(a.channels, CONV_V);
    int cx = 16;
    while (cx < 256 && cx < nv) cx *= 2;
    // narrower where that leaves fewer threads without a channel (4352 channels, 16 k rows: 64 side by side 57 us, 256 59 us; 32 no better)
    while (cx > 64 && cdiv(nv, cx / 2) * (cx / 2) < cdiv(nv, cx) * cx) cx /= 2;
    // longer runs read fewer rows twice; shorter ones give every CU several workgroups
    const Rows rows = {a.d_cu_seqlens, a.d_valid, a.batch, a.t};
    int R = 32;
    while (R > 8 && tiles_of(rows, R * (256 / cx)) * cdiv(nv, cx) < 2048) R /= 2;
    const long long grid = tiles_of(rows, R * (256 / cx)) * cdiv(nv, cx);
    MB_REQUIRE(launchable(grid, 256), "causal_conv1d: %d rows of %d channels are too many for one launch", a.t, a.channels);
    if (const int rc = conv_apart("causal_conv1d", a, false)) return rc;
    hipLaunchKernelGGL((causal_conv1d_kernel<T, K>), dim3((unsigned)grid), dim3(256), 0, s, a, cx, R);
  }
  MB_HIP(hipGetLastError());
  return MB_OK;
}

template <typename T> int conv_by_taps(const mb_causal_conv1d_args& a, bool step, hipStream_t s) {
  switch (a.ksize) {
    case 2: return launch_conv<T, 2>(a, step, s);
    case 3: return launch_conv<T, 3>(a, step, s);
    case 4: return launch_conv<T, 4>(a, step, s);
    case 5: return launch_conv<T, 5>(a, step, s);
    case 6: return launch_conv<T, 6>(a, step, s);
    case 7: return launch_conv<T, 7>(a, step, s);
    default: return launch_conv<T, 8>(a, step, s);
  }
}

static int check_conv(const char* name, const mb_causal_conv1d_args* a, bool step) {
  MB_REQUIRE(a, "%s: null arguments", name);
  MB_REQUIRE(a->dtype == MB_F32 || a->dtype == MB_F16 || a->dtype == MB_BF16, "%s: dtype %d is none of MB_F32, MB_F16, MB_BF16", name, a->dtype);
  MB_REQUIRE(a->ksize >= 2 && a->ksize <= 8, "%s: ksize %d is outside 2..8", name, a->ksize);
  MB_REQUIRE(a->act == 0 || a->act == 1, "%s: act %d is neither 0 (none) nor 1 (silu)", name, a->act);
  MB_REQUIRE(a->batch >= 0 && a->channels >= 0 && (step || a->t >= 0), "%s: negative shape", name);
  if (a->batch == 0 || a->channels == 0) return MB_OK;
  MB_REQUIRE(a->d_w, "%s: no weight", name);
  MB_REQUIRE((a->d_x && a->d_y) || (!step && a->t == 0), "%s: null x or y", name);
  MB_REQUIRE(!step || a->d_state, "%s: a step needs a state pool", name);
  if (a->d_state) {
    MB_REQUIRE(a->n_slots >= 0 && a->state_stride >= 0, "%s: negative state pool", name);
    MB_REQUIRE(a->d_slots || a->batch <= a->n_slots, "%s: %d items without slot numbers, but %d slots", name, a->batch, a->n_slots);
  } else {
    MB_REQUIRE(!a->d_slots && !a->d_has_state, "%s: slots or has_state without a state pool", name);
  }
  MB_REQUIRE(!a->d_cu_seqlens || !a->d_valid, "%s: packed and padded rows at once", name);
  MB_REQUIRE(step || (a->t <= 1 << 30 && a->batch <= 1 << 30), "%s: %d rows of %d items are too many", name, a->t, a->batch);
  return 1;
}

static int run_conv(const char* name, const mb_causal_conv1d_args* a, bool step, mb_stream_t stream) {
  const int go = check_conv(name, a, step);
  if (go <= 0) return go;
  if (a->dtype == MB_F32) return conv_by_taps<float>(*a, step, (hipStream_t)stream);
  if (a->dtype == MB_F16) return conv_by_taps<f16>(*a, step, (hipStream_t)stream);
  return conv_by_taps<bf16>(*a, step, (hipStream_t)stream);
}

}  // namespace ssm
}  // namespace mb

extern "C" int mb_causal_conv1d(const mb_causal_conv1d_args* a, mb_stream_t stream) { return mb::ssm::run_conv("causal_conv1d", a, false, stream); }
extern "C" int mb_causal_conv1d_step(const mb_causal_conv1d_args* a, mb_stream_t stream) {
  return mb::ssm::run_conv("causal_conv1d_step", a, true, stream);
}
