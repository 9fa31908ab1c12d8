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

// One pass over memory: a row (or, where the first norm's groups are all that couples channels, one group of a row) is held in
// registers, VPT vectors of 16 bytes per thread, by one wave (WAVE: up to 64 vectors, no barrier, 4 rows per workgroup) or one workgroup.
// Statistics are two-pass (mean, then centred squares) in fp32.  Memory-bound: 16384 x 4096 bf16 in 8 gated groups (6 bytes per element)
// takes 86 us (at best 83), 4.7 TB/s, of 5.2 that a large copy reaches; 8192 x 2048 bf16 with an fp32 residual (12 bytes) 36 us, warm.
// Why these widths: a wave with 4 vectors per lane holds 162 registers and ran that second case in 46 us; one vector per thread in
// workgroups of more than 256 threads loses to two (3001 fp16 channels: 46 and 41 us) unless there are too few rows to fill the chip
// (64 rows of 4096: 6.2 and 7.6 us); four vectors of a 16-bit type spill at 1024 threads, so they begin where two end.
template <typename T, typename TR, int VPT, bool WAVE>
__global__ __launch_bounds__(WAVE ? 256 : 1024) void block_norm_kernel(const mb_block_norm_args a, int parts, long long units) {
  constexpr bool FAST = sizeof(T) == 2;
  constexpr int V = 16 / sizeof(T);
  __shared__ float part[16];
  extern __shared__ float grouped[];  // groups with a next norm: a sum per vector, then mean and 1 / deviation per group
  const int tid = WAVE ? (int)threadIdx.x & 63 : (int)threadIdx.x, width = WAVE ? 64 : (int)blockDim.x, waves = WAVE ? 1 : width / 64;
  const long long unit = WAVE ? (long long)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (WAVE && unit >= units) return;
  const long long row = unit / parts;
  const int C = a.channels / parts, off = (int)(unit - row * parts) * C;
  const T* x = (const T*)a.d_x + row * a.x_rstride + off;
  const T* gate = a.d_gate ? (const T*)a.d_gate + row * a.gate_rstride + off : nullptr;
  const TR* res = a.d_residual ? (const TR*)a.d_residual + row * a.residual_rstride + off : nullptr;
  const float inv_c = 1.f / C;
  auto column = [&](int i) { return (i * width + tid) * V; };

  Vec<T, V> xr[VPT], gr[VPT];
  Vec<TR, V> rr[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {  // everything is requested before anything is used
    const int c = column(i), n = C - c;
    xr[i] = load_some<T, V>(x + c, n);
    if (gate) gr[i] = load_some<T, V>(gate + c, n);
    if (res) rr[i] = load_some<TR, V>(res + c, n);
  }
  float v[VPT][V];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      v[i][k] = to_f32(xr[i].v[k]);
      if (gate && a.gate_first) v[i][k] *= gate_of<FAST>(to_f32(gr[i].v[k]), a.gate_act);
    }
  // mean and 1 / deviation of the row in registers; columns beyond the row do not count
  auto statistics = [&](int kind, float eps, float& mean, float& inv) {
    mean = 0.f;
    if (kind == 2) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) mean += column(i) + k < C ? v[i][k] : 0.f;
      mean = block_sum(mean, part, waves) * inv_c;
    }
    float m2 = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float d = column(i) + k < C ? v[i][k] - mean : 0.f;
        m2 = fmaf(d, d, m2);
      }
    inv = 1.f / sqrtf(block_sum(m2, part, waves) * inv_c + eps);
  };
  auto affine = [&](const float* w, const float* b, int i) {
    const int c = column(i), n = C - c;
    if (w) {
      const Vec<float, V> t = load_some<float, V>(w + off + c, n);
#pragma unroll
      for (int k = 0; k < V; ++k) v[i][k] *= t.v[k];
    }
    if (b) {
      const Vec<float, V> t = load_some<float, V>(b + off + c, n);
#pragma unroll
      for (int k = 0; k < V; ++k) v[i][k] += t.v[k];
    }
  };
  if (a.norm) {
    if (WAVE || a.groups == parts) {
      float mean, inv;
      statistics(a.norm, a.eps, mean, inv);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) v[i][k] = (v[i][k] - mean) * inv;
    } else {  // several groups in this row: V divides a group, every vector belongs to one
      const int gs = C / a.groups, gv = gs / V, nv = C / V;
      float* stat = grouped + nv;
      for (int pass = a.norm == 2 ? 0 : 1; pass < 2; ++pass) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int c = column(i);
          if (c >= C) continue;
          const float mean = a.norm == 2 && pass ? stat[2 * (c / gs)] : 0.f;
          float s = 0.f;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const float d = v[i][k] - mean;
            s = pass ? fmaf(d, d, s) : s + d;
          }
          grouped[c / V] = s;
        }
        __syncthreads();
        for (int g = tid >> 6; g < a.groups; g += waves) {
          float s = 0.f;
          for (int j = tid & 63; j < gv; j += 64) s += grouped[g * gv + j];
          s = wave_sum(s) / gs;
          if ((tid & 63) == 0) stat[2 * g + pass] = pass ? 1.f / sqrtf(s + a.eps) : s;
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = column(i);
        if (c >= C) continue;
        const float mean = a.norm == 2 ? stat[2 * (c / gs)] : 0.f, inv = stat[2 * (c / gs) + 1];
#pragma unroll
        for (int k = 0; k < V; ++k) v[i][k] = (v[i][k] - mean) * inv;
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) affine(a.d_weight, a.d_bias, i);
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = column(i), n = C - c;
    if (gate && !a.gate_first) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[i][k] *= gate_of<FAST>(to_f32(gr[i].v[k]), a.gate_act);
    }
    if (a.d_scale) {
      const Vec<float, V> t = load_some<float, V>(a.d_scale + off + c, n);
#pragma unroll
      for (int k = 0; k < V; ++k) v[i][k] *= a.res_scale * t.v[k];
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) v[i][k] *= a.res_scale;
    }
    if (res) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[i][k] += to_f32(rr[i].v[k]);
    }
    if (a.d_sum) {
      Vec<TR, V> o;
#pragma unroll
      for (int k = 0; k < V; ++k) o.v[k] = from_f32<TR>(v[i][k]);
      store_some<TR, V>((TR*)a.d_sum + row * a.sum_rstride + off + c, o, n);
    }
  }
  if (!a.next_norm) return;
  float mean, inv;
  statistics(a.next_norm, a.next_eps, mean, inv);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = column(i), n = C - c;
#pragma unroll
    for (int k = 0; k < V; ++k) v[i][k] = (v[i][k] - mean) * inv;
    affine(a.d_next_weight, a.d_next_bias, i);
    Vec<T, V> o;
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = from_f32<T>(v[i][k]);
    store_some<T, V>((T*)a.d_y + row * a.y_rstride + off + c, o, n);
  }
}

// Any width, groups of any size: one workgroup per row, three passes over the row, element by element.  Rows that registers hold come here
// only for groups that no number of 16-byte vectors fills, with a next norm: 8192 x 2000 bf16, 4 groups, gate, fp32 residual, next norm take
// 152 us where 2048 channels take 41.
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
  constexpr int V = 16 / sizeof(T);
  // groups couple nothing but themselves without a next norm: each is a row of its own
  const int parts = a.next_norm ? 1 : a.groups, C = a.channels / parts, nv = cdiv(C, V);
  const long long units = a.rows * parts;
  const bool grouped = a.groups != parts;
  const bool wave = !grouped && nv <= 64;
  const bool whole = nv <= 4096 && (!grouped || (C / a.groups) % V == 0) && units < (1ll << 31);
  const size_t lds = whole && !wave && grouped ? ((size_t)nv + 2 * a.groups) * sizeof(float) : 0;
  const int vpt = nv <= (units < 512 ? 1024 : 256) ? 1 : nv <= 2048 ? 2 : 4, threads = wave || !whole ? 256 : (cdiv(nv, vpt) + 63) / 64 * 64;
  const long long grid = !whole ? a.rows : wave ? (units + 3) / 4 : units;
  MB_REQUIRE(launchable(grid, threads), "block_norm: %lld rows of %d channels are too many for one launch", a.rows, a.channels);
#define MB_NORM(VPT, WAVE) hipLaunchKernelGGL((block_norm_kernel<T, TR, VPT, WAVE>), dim3((unsigned)grid), dim3(threads), lds, s, a, parts, units)
  if (whole && wave) {
    MB_NORM(1, true);
  } else if (whole) {
    if (vpt == 1) MB_NORM(1, false);
    else if (vpt == 2) MB_NORM(2, false);
    else MB_NORM(4, false);
  } else {
    hipLaunchKernelGGL((block_norm_row_kernel<T, TR>), dim3((unsigned)grid), dim3(threads), (size_t)2 * a.groups * sizeof(float), s, a);
  }
#undef MB_NORM
  MB_HIP(hipGetLastError());
  return MB_OK;
}

// An output is exactly one of x, gate and residual (a thread reads an element before it writes it), or overlaps nothing.
static int norm_apart(const mb_block_norm_args& a) {
  const size_t e = size_of(a.dtype), r = size_of(a.res_dtype);
  const Span s[] = {span_of("the sum", a.d_sum, r, a.channels, a.rows, a.sum_rstride),
                    span_of("out", a.d_y, e, a.channels, a.rows, a.y_rstride),
                    span_of("weight", a.d_weight, 4, a.channels),
                    span_of("bias", a.d_bias, 4, a.channels),
                    span_of("scale", a.d_scale, 4, a.channels),
                    span_of("next_weight", a.d_next_weight, 4, a.channels),
                    span_of("next_bias", a.d_next_bias, 4, a.channels),
                    span_of("x", a.d_x, e, a.channels, a.rows, a.x_rstride),
                    span_of("gate", a.d_gate, e, a.channels, a.rows, a.gate_rstride),
                    span_of("residual", a.d_residual, r, a.channels, a.rows, a.residual_rstride)};
  return check_apart("block_norm", s, 2, 10, 7);
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
  if (const int rc = norm_apart(*a)) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (a->dtype == MB_F32) return launch_norm<float, float>(*a, s);
  if (a->dtype == MB_F16) return a->res_dtype == MB_F32 ? launch_norm<f16, float>(*a, s) : launch_norm<f16, f16>(*a, s);
  return a->res_dtype == MB_F32 ? launch_norm<bf16, float>(*a, s) : launch_norm<bf16, bf16>(*a, s);
}
