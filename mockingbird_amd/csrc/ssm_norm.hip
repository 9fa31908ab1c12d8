// The seam between two blocks of a residual network: gate, norm of the block's output, residual scale and sum, norm of the next block.
#include "ssm.h"

namespace mb {
namespace ssm {

template <bool FAST> __device__ __forceinline__ float gate_of(float g, int act) {
  return act == 1 ? g * sigmoid<FAST>(g) : act == 2 ? sigmoid<FAST>(g) : g;
}

__device__ __forceinline__ float block_sum(float v, float* part, int waves) {  // every thread gets the sum, in one fixed order
  v = wave_sum(v);
  if (waves == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < waves; ++i) v += part[i];
  return v;
}

// Any width: one workgroup per row, three passes over the row.  Statistics are two-pass (mean, then centred squares) in fp32.
template <typename T, typename TR>
__global__ __launch_bounds__(256) void block_norm_row_kernel(const mb_block_norm_args a) {
  constexpr bool FAST = sizeof(T) == 2;
  extern __shared__ float stats[];  // [groups][2] mean, 1 / deviation of the first norm
  __shared__ float part[4];
  const long long row = blockIdx.x;
  const T* x = (const T*)a.d_x + row * a.x_rstride;
  const T* gate = a.d_gate ? (const T*)a.d_gate + row * a.gate_rstride : nullptr;
  const TR* res = a.d_residual ? (const TR*)a.d_residual + row * a.residual_rstride : nullptr;
  TR* sum = a.d_sum ? (TR*)a.d_sum + row * a.sum_rstride : nullptr;
  T* y = a.d_y ? (T*)a.d_y + row * a.y_rstride : nullptr;
  const int gs = a.channels / a.groups;
  auto in = [&](int c) {
    float v = to_f32(x[c]);
    if (gate && a.gate_first) v *= gate_of<FAST>(to_f32(gate[c]), a.gate_act);
    return v;
  };
  for (int g = 0; g < (a.norm ? a.groups : 0); ++g) {
    float mean = 0.f, m2 = 0.f;
    if (a.norm == 2) {
      for (int c = threadIdx.x; c < gs; c += 256) mean += in(g * gs + c);
      mean = block_sum(mean, part, 4) / gs;
    }
    for (int c = threadIdx.x; c < gs; c += 256) {
      const float d = in(g * gs + c) - mean;
      m2 = fmaf(d, d, m2);
    }
    m2 = block_sum(m2, part, 4);
    if (threadIdx.x == 0) stats[2 * g] = mean, stats[2 * g + 1] = 1.f / sqrtf(m2 / gs + a.eps);
  }
  __syncthreads();
  auto total = [&](int c) {
    float v = in(c);
    if (a.norm) {
      v = (v - stats[2 * (c / gs)]) * stats[2 * (c / gs) + 1];
      if (a.d_weight) v *= a.d_weight[c];
      if (a.d_bias) v += a.d_bias[c];
    }
    if (gate && !a.gate_first) v *= gate_of<FAST>(to_f32(gate[c]), a.gate_act);
    v *= a.d_scale ? a.res_scale * a.d_scale[c] : a.res_scale;
    return res ? v + to_f32(res[c]) : v;
  };
  float mean = 0.f, inv = 1.f;
  if (a.next_norm) {
    float m2 = 0.f;
    if (a.next_norm == 2) {
      for (int c = threadIdx.x; c < a.channels; c += 256) mean += total(c);
      mean = block_sum(mean, part, 4) / a.channels;
    }
    for (int c = threadIdx.x; c < a.channels; c += 256) {
      const float d = total(c) - mean;
      m2 = fmaf(d, d, m2);
    }
    inv = 1.f / sqrtf(block_sum(m2, part, 4) / a.channels + a.next_eps);
  }
  for (int c = threadIdx.x; c < a.channels; c += 256) {  // each thread has read an element before it writes that element's outputs
    const float v = total(c);
    if (sum) sum[c] = from_f32<TR>(v);
    if (a.next_norm) {
      float o = (v - mean) * inv;
      if (a.d_next_weight) o *= a.d_next_weight[c];
      if (a.d_next_bias) o += a.d_next_bias[c];
      y[c] = from_f32<T>(o);
    }
  }
}

template <typename T, typename TR> int launch_norm(const mb_block_norm_args& a, hipStream_t s) {
  hipLaunchKernelGGL((block_norm_row_kernel<T, TR>), dim3((unsigned)a.rows), dim3(256), (size_t)2 * a.groups * sizeof(float), s, a);
  MB_HIP(hipGetLastError());
  return MB_OK;
}

static int check_norm(const mb_block_norm_args* a) {
  MB_REQUIRE(a, "block_norm: null arguments");
  MB_REQUIRE(a->dtype == MB_F32 || a->dtype == MB_F16 || a->dtype == MB_BF16, "block_norm: dtype %d is none of MB_F32, MB_F16, MB_BF16", a->dtype);
  MB_REQUIRE(a->res_dtype == a->dtype || a->res_dtype == MB_F32, "block_norm: res_dtype %d is neither dtype nor MB_F32", a->res_dtype);
  MB_REQUIRE(a->norm >= 0 && a->norm <= 2 && a->next_norm >= 0 && a->next_norm <= 2, "block_norm: norm kinds are 0, 1 (RMS), 2 (layer)");
  MB_REQUIRE(a->gate_act >= 0 && a->gate_act <= 2, "block_norm: gate_act %d is outside 0..2", a->gate_act);
  MB_REQUIRE(a->rows >= 0 && a->channels >= 0, "block_norm: negative shape");
  MB_REQUIRE(a->groups >= 1 && a->groups <= 1024 && a->channels % a->groups == 0, "block_norm: %d channels in %d groups (1..1024 equal ones)",
             a->channels, a->groups);
  MB_REQUIRE(a->norm || a->groups == 1, "block_norm: groups without a first norm");
  MB_REQUIRE(a->norm || a->next_norm || a->d_residual || a->d_gate, "block_norm: nothing to compute");
  MB_REQUIRE(a->rows < (1ll << 31), "block_norm: %lld rows are too many for one launch", a->rows);
  if (a->rows == 0 || a->channels == 0) return MB_OK;
  MB_REQUIRE(a->d_x, "block_norm: null x");
  MB_REQUIRE(a->next_norm ? a->d_y != nullptr : a->d_sum && !a->d_y, "block_norm: y comes with next_norm and only then; without it sum is the result");
  return 1;
}

}  // namespace ssm
}  // namespace mb

extern "C" int mb_block_norm(const mb_block_norm_args* a, mb_stream_t stream) {
  using namespace mb::ssm;
  const int go = check_norm(a);
  if (go <= 0) return go;
  hipStream_t s = (hipStream_t)stream;
  if (a->dtype == MB_F32) return launch_norm<float, float>(*a, s);
  if (a->dtype == MB_F16) return a->res_dtype == MB_F32 ? launch_norm<f16, float>(*a, s) : launch_norm<f16, f16>(*a, s);
  return a->res_dtype == MB_F32 ? launch_norm<bf16, float>(*a, s) : launch_norm<bf16, bf16>(*a, s);
}
