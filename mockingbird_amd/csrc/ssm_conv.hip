// Short causal depthwise convolution over rows of channels, with the last inputs of every item kept as its state.
//   y[t][c] = act(bias[c] + sum_j w[c][j] x[t - K + 1 + j][c])
#include "ssm.h"

namespace mb {
namespace ssm {

template <typename T, int K, int V>
__global__ __launch_bounds__(256) void causal_conv1d_kernel(const mb_causal_conv1d_args a, int cx, int R) {
  constexpr bool FAST = sizeof(T) == 2;
  const int ci = threadIdx.x & (cx - 1), rg = threadIdx.x / cx, groups = 256 / cx;
  const int blocks_c = (a.channels + cx * V - 1) / (cx * V);
  const unsigned tile = blockIdx.x / blocks_c;
  const int c = ((int)(blockIdx.x - tile * blocks_c) * cx + ci) * V;
  const Rows rows = {a.d_cu_seqlens, a.d_valid, a.batch, a.t};
  const Item it = item_of(rows, tile, R * groups);
  if (it.part < 0 || it.part >= max(1, (it.len + R * groups - 1) / (R * groups))) return;
  int slot = -1;
  if (a.d_state) {
    slot = slot_of(a.d_slots, it.b, a.n_slots);
    if (slot < 0) return;
  }
  if (c >= a.channels) return;
  const T* x = (const T*)a.d_x + it.row * a.x_rstride + (a.d_cu_seqlens ? 0 : it.b * a.x_bstride) + c;
  T* y = (T*)a.d_y + it.row * a.y_rstride + (a.d_cu_seqlens ? 0 : it.b * a.y_bstride) + c;
  float w[V][K], bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j < K; ++j) w[i][j] = a.d_w[(long long)(c + i) * K + j];
    bias[i] = a.d_bias ? a.d_bias[c + i] : 0.f;
  }
  const int t0 = (it.part * groups + rg) * R, t1 = min(it.len, t0 + R);
  Vec<T, V> win[K - 1];  // rows t - K + 1 .. t - 1
  const bool first = it.part == 0 && rg == 0;
  if (first) {
    T* st = a.d_state ? (T*)a.d_state + slot * a.state_stride + c : nullptr;
    const bool keep = st && (!a.d_has_state || a.d_has_state[it.b]);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      if (keep) win[j] = load_vec<T, V>(st + (long long)j * a.channels);
      else
        for (int i = 0; i < V; ++i) win[j].v[i] = (T)0.f;
    }
    if (st) {  // only this thread touches these channels of the slot: the old rows are in registers before the new ones are written
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        const int from = it.len + j;  // row of (state ++ x): the last K - 1 of it
        Vec<T, V> v;
        if (from >= K - 1) v = load_vec<T, V>(x + (from - (K - 1)) * a.x_rstride);
        else {
#pragma unroll
          for (int k = 0; k < K - 1; ++k)
            if (k == from) v = win[k];
        }
        store_vec<T, V>(st + (long long)j * a.channels, v);
      }
    }
  } else if (t0 < t1) {  // R >= K - 1: these rows are the item's own
#pragma unroll
    for (int j = 0; j < K - 1; ++j) win[j] = load_vec<T, V>(x + (t0 - (K - 1) + j) * a.x_rstride);
  }
  for (int t = t0; t < t1; ++t) {
    const Vec<T, V> cur = load_vec<T, V>(x + t * a.x_rstride);
    Vec<T, V> out;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = bias[i];
#pragma unroll
      for (int j = 0; j < K - 1; ++j) v = fmaf(w[i][j], to_f32(win[j].v[i]), v);
      v = fmaf(w[i][K - 1], to_f32(cur.v[i]), v);
      if (a.act) v *= sigmoid<FAST>(v);
      out.v[i] = from_f32<T>(v);
    }
    store_vec<T, V>(y + t * a.y_rstride, out);
#pragma unroll
    for (int j = 0; j + 1 < K - 1; ++j) win[j] = win[j + 1];
    win[K - 2] = cur;
  }
}

// One row per item: the same sum with the state as the window; the state moves up by one row in place.
template <typename T, int K, int V>
__global__ __launch_bounds__(64) void causal_conv1d_step_kernel(const mb_causal_conv1d_args a) {
  constexpr bool FAST = sizeof(T) == 2;
  const int per = (a.channels + 64 * V - 1) / (64 * V);
  const int b = (int)(blockIdx.x / per);
  const int c = ((int)(blockIdx.x - (unsigned)b * per) * 64 + (int)threadIdx.x) * V;
  const int slot = slot_of(a.d_slots, b, a.n_slots);
  if (slot < 0 || c >= a.channels) return;
  const Vec<T, V> cur = load_vec<T, V>((const T*)a.d_x + b * a.x_rstride + c);
  T* st = (T*)a.d_state + slot * a.state_stride + c;
  Vec<T, V> win[K - 1], out;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) win[j] = load_vec<T, V>(st + (long long)j * a.channels);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float* w = a.d_w + (long long)(c + i) * K;
    float v = a.d_bias ? a.d_bias[c + i] : 0.f;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) v = fmaf(w[j], to_f32(win[j].v[i]), v);
    v = fmaf(w[K - 1], to_f32(cur.v[i]), v);
    if (a.act) v *= sigmoid<FAST>(v);
    out.v[i] = from_f32<T>(v);
  }
  store_vec<T, V>((T*)a.d_y + b * a.y_rstride + c, out);
#pragma unroll
  for (int j = 0; j + 1 < K - 1; ++j) store_vec<T, V>(st + (long long)j * a.channels, win[j + 1]);
  store_vec<T, V>(st + (long long)(K - 2) * a.channels, cur);
}

template <typename T, int K, int V> int launch_conv(const mb_causal_conv1d_args& a, bool step, hipStream_t s) {
  const int nv = (a.channels + V - 1) / V;
  if (step) {
    const long long grid = (long long)a.batch * ((nv + 63) / 64);
    MB_REQUIRE(grid < (1ll << 31), "causal_conv1d_step: %d items of %d channels are too many for one launch", a.batch, a.channels);
    hipLaunchKernelGGL((causal_conv1d_step_kernel<T, K, V>), dim3((unsigned)grid), dim3(64), 0, s, a);
  } else {
    int cx = 16;
    while (cx < 256 && cx < nv) cx *= 2;
    const int R = 16, groups = 256 / cx;
    const Rows rows = {a.d_cu_seqlens, a.d_valid, a.batch, a.t};
    const long long grid = tiles_of(rows, R * groups) * ((nv + cx - 1) / cx);
    MB_REQUIRE(grid < (1ll << 31), "causal_conv1d: %d rows of %d channels are too many for one launch", a.t, a.channels);
    hipLaunchKernelGGL((causal_conv1d_kernel<T, K, V>), dim3((unsigned)grid), dim3(256), 0, s, a, cx, R);
  }
  MB_HIP(hipGetLastError());
  return MB_OK;
}

template <typename T, int V> int conv_by_taps(const mb_causal_conv1d_args& a, bool step, hipStream_t s) {
  switch (a.ksize) {
    case 2: return launch_conv<T, 2, V>(a, step, s);
    case 3: return launch_conv<T, 3, V>(a, step, s);
    case 4: return launch_conv<T, 4, V>(a, step, s);
    case 5: return launch_conv<T, 5, V>(a, step, s);
    case 6: return launch_conv<T, 6, V>(a, step, s);
    case 7: return launch_conv<T, 7, V>(a, step, s);
    default: return launch_conv<T, 8, V>(a, step, s);
  }
}

template <typename T> int conv_by_width(const mb_causal_conv1d_args& a, bool step, hipStream_t s) {
  constexpr int WIDE = 16 / sizeof(T);
  // 16 bytes per access where every row of every tensor keeps that alignment; otherwise one element
  const long long all = a.channels | a.x_rstride | a.y_rstride | (step || a.d_cu_seqlens ? 0 : a.x_bstride | a.y_bstride) |
                        (a.d_state ? a.state_stride : 0);
  if (all % WIDE == 0 && aligned(a.d_x, 16) && aligned(a.d_y, 16) && aligned(a.d_state, 16)) return conv_by_taps<T, WIDE>(a, step, s);
  return conv_by_taps<T, 1>(a, step, s);
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
  MB_REQUIRE(!a->d_cu_seqlens || (long long)a->t + a->batch < (1ll << 31), "%s: %d rows of %d items are too many", name, a->t, a->batch);
  return 1;
}

static int run_conv(const char* name, const mb_causal_conv1d_args* a, bool step, mb_stream_t stream) {
  const int go = check_conv(name, a, step);
  if (go <= 0) return go;
  if (a->dtype == MB_F32) return conv_by_width<float>(*a, step, (hipStream_t)stream);
  if (a->dtype == MB_F16) return conv_by_width<f16>(*a, step, (hipStream_t)stream);
  return conv_by_width<bf16>(*a, step, (hipStream_t)stream);
}

}  // namespace ssm
}  // namespace mb

extern "C" int mb_causal_conv1d(const mb_causal_conv1d_args* a, mb_stream_t stream) { return mb::ssm::run_conv("causal_conv1d", a, false, stream); }
extern "C" int mb_causal_conv1d_step(const mb_causal_conv1d_args* a, mb_stream_t stream) {
  return mb::ssm::run_conv("causal_conv1d_step", a, true, stream);
}
