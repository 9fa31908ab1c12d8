// Selective state space scan: per head a state h [head_dim][d_state] that decays by exp(d A), takes in (d x) B^T and answers y = h C + D x.
#include "ssm_scan_chunk.h"

namespace mb {
namespace ssm {

template <int LANES> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// One row per item: the state is read and written once (8 bytes per element of it), which is all that counts with many items.  LANES
// lanes hold a state row (4 columns each), 256 / LANES rows at a time; a workgroup takes `pb` rows of one head, U passes requested at once.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void selective_scan_step_kernel(const mb_selective_scan_args a, int pb) {
  constexpr int ROWS = 256 / LANES, U = 4;
  const int splits = (a.head_dim + pb - 1) / pb;
  const unsigned item_head = blockIdx.x / splits;
  const int p0 = (int)(blockIdx.x - item_head * splits) * pb;
  const int b = (int)(item_head / a.heads), head = (int)(item_head - (unsigned)b * a.heads);
  const int slot = slot_of(a.d_slots, b, a.n_slots);
  if (slot < 0) return;
  const int n = (int)(threadIdx.x % LANES) * 4, left = a.d_state_dim - n;
  const int group = head / (a.heads / a.groups);
  const int p1 = min(a.head_dim, p0 + pb);
  float* h = a.d_state + slot * a.state_stride + (long long)head * a.head_dim * a.d_state_dim + n;
  const T* x = (const T*)a.d_x + b * a.x_rstride + (long long)head * a.head_dim;
  T* y = (T*)a.d_y + b * a.y_rstride + (long long)head * a.head_dim;
  float decay = 0.f, d = 0.f;
  Vec<T, 4> br, cr;
  const float skip = a.d_d ? a.d_d[head] : 0.f;
  for (int q = p0; q < p1; q += U * ROWS) {
    const int p = q + (int)threadIdx.x / LANES;
    Vec<float, 4> v[U];
    float xv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = p + u * ROWS;
      v[u] = load_some<float, 4>(h + (long long)r * a.d_state_dim, r < p1 ? left : 0);
      xv[u] = r < p1 ? to_f32(x[r]) : 0.f;
    }
    if (q == p0) {  // behind the first states' requests
      br = load_some<T, 4>((const T*)a.d_b + b * a.b_rstride + (long long)group * a.d_state_dim + n, left);
      cr = load_some<T, 4>((const T*)a.d_c + b * a.c_rstride + (long long)group * a.d_state_dim + n, left);
      d = step_size(a, b * a.dt_rstride + head, head);
      decay = expf(d * a.d_a[head]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = p + u * ROWS;
      const float dx = d * xv[u];
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float next = fmaf(v[u].v[i], decay, dx * to_f32(br.v[i]));
        v[u].v[i] = i < left ? next : 0.f;  // (0 * infinity in columns that are not there)
        s = fmaf(v[u].v[i], to_f32(cr.v[i]), s);
      }
      s = lanes_sum<LANES>(s);
      if (r < p1) {
        store_some<float, 4>(h + (long long)r * a.d_state_dim, v[u], left);
        if (n == 0) y[r] = from_f32<T>(fmaf(skip, xv[u], s));
      }
    }
  }
}

// Between the two passes of a split call: what every tile adds becomes the state in front of the next one.  A workgroup takes 1024 elements
// of a head of the j-th item that is split, 4 per thread; the tiles are read U ahead of the chain that runs over them.
__global__ __launch_bounds__(256) void selective_scan_join_kernel(const mb_selective_scan_args a, const Split sp) {
  constexpr int U = 4;
  const int elems = a.head_dim * a.d_state_dim, blocks = (elems + 1023) / 1024;
  const unsigned item_head = blockIdx.x / blocks;
  const int e = ((int)(blockIdx.x - item_head * blocks) * 256 + (int)threadIdx.x) * 4, n = elems - e;
  const int j = (int)(item_head / a.heads), head = (int)(item_head - (unsigned)j * a.heads);
  const Rows rows = {a.d_cu_seqlens, a.d_valid, a.batch, a.t};
  const Long it = long_item(rows, j, sp.seg);
  if (it.b < 0) return;
  int slot = -1;
  if (a.d_state) {
    slot = slot_of(a.d_slots, it.b, a.n_slots);
    if (slot < 0) return;
  }
  const bool keep = a.d_state && (!a.d_has_state || a.d_has_state[it.b]);
  const int at = keep ? initial_at(sp, a.batch, it.b, it.fronts) : 0;
  if (n <= 0 || at < 0 || it.fronts > sp.fronts - (it.parts - 1)) return;  // (row numbers that overlap can claim more tiles than there are)
  Vec<float, 4> h = load_some<float, 4>(a.d_state + slot * a.state_stride + (long long)head * elems + e, keep ? n : 0);
  const long long step = (long long)a.heads * elems, own_head = (long long)head * elems + e;
  if (keep) store_some<float, 4>(sp.initial + at * step + own_head, h, n);
  float* st = sp.state + it.fronts * step + own_head;
  const float* decay = sp.decay + (long long)it.fronts * a.heads + head;
  for (int k = 1; k < it.parts; k += U) {
    Vec<float, 4> own[U];
    float by[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      own[u] = load_some<float, 4>(st + u * step, k + u < it.parts ? n : 0);
      by[u] = k + u < it.parts ? decay[(long long)u * a.heads] : 0.f;
    }
    const Vec<float, 4> was = h;
    bool spoilt = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) h.v[i] = fmaf(h.v[i], by[u], own[u].v[i]);
      if (k + u < it.parts) store_some<float, 4>(st + u * step, h, n);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) spoilt |= isnan(h.v[i]);
    if (__builtin_expect(spoilt, 0)) {
      // The decay of a whole tile can leave fp32 where no row's does (-0: one does): what is infinite stays so beside a zero, a zero beside an
      // infinity.
      h = was;
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = h.v[i] * by[u];
          if (isnan(v) && !isnan(h.v[i]) && !isnan(by[u]) && __float_as_uint(by[u]) != 0x80000000u) v = h.v[i];
          h.v[i] = v + own[u].v[i];
        }
        if (k + u < it.parts) store_some<float, 4>(st + u * step, h, n);
      }
    }
    st += U * step;
    decay += (long long)U * a.heads;
  }
}

template <typename T, int LANES> int launch_step(const mb_selective_scan_args& a, hipStream_t s) {
  constexpr int ROWS = 256 / LANES;
  int pb = (a.head_dim + ROWS - 1) / ROWS * ROWS;
  // few requests: a head's rows are dealt to more workgroups, down to one pass each, until two fit every CU
  while (pb > ROWS && (long long)a.batch * a.heads * ((a.head_dim + pb - 1) / pb) < 512) pb = (pb / ROWS + 1) / 2 * ROWS;
  const long long grid = (long long)a.batch * a.heads * ((a.head_dim + pb - 1) / pb);
  MB_REQUIRE(launchable(grid, 256), "selective_scan_step: %d items of %d heads are too many for one launch", a.batch, a.heads);
  hipLaunchKernelGGL((selective_scan_step_kernel<T, LANES>), dim3((unsigned)grid), dim3(256), 0, s, a, pb);
  MB_HIP(hipGetLastError());
  return MB_OK;
}

template <typename T> int step_by_lanes(const mb_selective_scan_args& a, hipStream_t s) {
  if (a.d_state_dim <= 16) return launch_step<T, 4>(a, s);
  if (a.d_state_dim <= 32) return launch_step<T, 8>(a, s);
  if (a.d_state_dim <= 64) return launch_step<T, 16>(a, s);
  if (a.d_state_dim <= 128) return launch_step<T, 32>(a, s);
  return launch_step<T, 64>(a, s);
}

// Rows of a time tile, or 0 for one workgroup walking a whole item.  Splitting costs a second pass over x and B, and states through memory;
// it pays where the items alone would leave CUs without a workgroup.  The host does not know the lengths of packed items: it deals out the
// rows of all together, and with enough items splits only those of more than twice the mean length.
static int rows_per_tile(const mb_selective_scan_args& a) {
  const long long units = (long long)a.groups * cdiv(a.heads / a.groups, 2) * cdiv(a.head_dim, 64);
  const long long all = a.d_cu_seqlens ? a.t : (long long)a.t * a.batch;
  const bool full = units * a.batch >= 256;
  // up to five chunks one walk is shorter than three launches (24 heads of 64 x 128 bf16: 256 rows 28 and 33 us, 384 rows 37 and 33 us)
  const int chunk = a.dtype == MB_BF16 && a.d_state_dim <= 128 ? 64 : 32;
  if ((full && !a.d_cu_seqlens) || a.t <= 5 * chunk) return 0;
  long long seg = (all * units + 511) / 512;  // two workgroups per CU
  // shorter tiles shorten the walk but move more states: not below 128 rows where a head's state outweighs 64 rows of its x
  const int least = a.head_dim * a.d_state_dim < 4096 ? 64 : 128;
  if (seg < least) seg = least;
  if (full && seg < 2 * all / a.batch) seg = 2 * all / a.batch;
  seg = (seg + 63) / 64 * 64;
  return seg >= a.t ? 0 : (int)seg;
}

static size_t split_layout(const mb_selective_scan_args& a, void* base, Split* sp) {
  *sp = {};
  sp->seg = rows_per_tile(a);
  if (!sp->seg) return 0;
  const Rows rows = {a.d_cu_seqlens, a.d_valid, a.batch, a.t};
  const long long fronts = fronts_of(rows, sp->seg), initials = a.d_state ? (a.batch < fronts ? a.batch : fronts) : 0;
  const size_t state = (size_t)a.heads * a.head_dim * a.d_state_dim;
  sp->fronts = (int)fronts;
  sp->initials = (int)initials;
  Arena ar(base, ~(size_t)0);
  sp->state = ar.take<float>(fronts * state);
  sp->initial = ar.take<float>(initials * state);
  sp->decay = ar.take<float>(fronts * a.heads);
  return align_up(ar.off, 256);
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
  MB_REQUIRE((long long)a->batch * a->heads < (1ll << 31) && (a->d_cu_seqlens || (long long)a->batch * (step ? 1 : a->t) < (1ll << 40)),
             "%s: %d items of %d rows and %d heads are too many for one launch", name, a->batch, a->t, a->heads);
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
  MB_REQUIRE(step || (a->t <= 1 << 30 && a->batch <= 1 << 30), "%s: %d rows of %d items are too many", name, a->t, a->batch);
  return 1;
}

static int scan_apart(const char* name, const mb_selective_scan_args& a, bool step, const void* ws, size_t ws_bytes) {
  const size_t e = size_of(a.dtype);
  const bool padded = !step && !a.d_cu_seqlens;
  const long long rows = step ? a.batch : a.t, items = padded ? a.batch : 1, wide = (long long)a.heads * a.head_dim, narrow = (long long)a.groups * a.d_state_dim;
  const Span s[] = {span_of("out", a.d_y, e, wide, rows, a.y_rstride, items, a.y_bstride),
                    span_of("state", a.d_state, 4, wide * a.d_state_dim, a.n_slots, a.state_stride),
                    span_of("the workspace", ws, 1, (long long)ws_bytes),
                    span_of("x", a.d_x, e, wide, rows, a.x_rstride, items, a.x_bstride),
                    span_of("dt", a.d_dt, size_of(a.dt_dtype), a.heads, rows, a.dt_rstride, items, a.dt_bstride),
                    span_of("B", a.d_b, e, narrow, rows, a.b_rstride, items, a.b_bstride),
                    span_of("C", a.d_c, e, narrow, rows, a.c_rstride, items, a.c_bstride),
                    span_of("A", a.d_a, 4, a.heads),
                    span_of("D", a.d_d, 4, a.heads),
                    span_of("dt_bias", a.d_dt_bias, 4, a.heads),
                    span_of("slots", a.d_slots, 4, a.batch),
                    span_of("has_state", step ? nullptr : a.d_has_state, 1, a.batch),
                    span_of("cu_seqlens", step ? nullptr : a.d_cu_seqlens, 4, a.batch + 1ll),
                    span_of("lengths", step ? nullptr : a.d_valid, 4, a.batch)};
  return check_apart(name, s, 3, sizeof(s) / sizeof(*s));
}

static int run_scan(const mb_selective_scan_args* a, void* ws, size_t ws_bytes, hipStream_t s) {
  const int go = check_scan("selective_scan", a, false);
  if (go <= 0) return go;
  Split sp;
  const size_t need = split_layout(*a, ws, &sp);
  if (ws_bytes < need || (need && !ws)) {
    set_error("selective_scan: workspace of %zu B, %zu B are needed", ws_bytes, need);
    return MB_ENOMEM;
  }
  MB_REQUIRE(aligned(ws, 16), "selective_scan: the workspace must be 16-byte aligned");
  if (const int rc = scan_apart("selective_scan", *a, false, ws, need)) return rc;
  auto* chunks = a->dtype == MB_F32 ? scan_chunks_f32 : a->dtype == MB_F16 ? scan_chunks_f16 : scan_chunks_bf16;
  if (sp.seg) {
    const int rc = chunks(*a, sp, true, s);
    if (rc) return rc;
    const long long grid = (long long)(a->batch < sp.fronts ? a->batch : sp.fronts) * a->heads * cdiv(a->head_dim * a->d_state_dim, 1024);
    MB_REQUIRE(launchable(grid, 256), "selective_scan: %d items of %d heads are too many for one launch", a->batch, a->heads);
    hipLaunchKernelGGL(selective_scan_join_kernel, dim3((unsigned)grid), dim3(256), 0, s, *a, sp);
    MB_HIP(hipGetLastError());
  }
  return chunks(*a, sp, false, s);
}

static int run_step(const mb_selective_scan_args* a, hipStream_t s) {
  const int go = check_scan("selective_scan_step", a, true);
  if (go <= 0) return go;
  if (const int rc = scan_apart("selective_scan_step", *a, true, nullptr, 0)) return rc;
  return a->dtype == MB_F32 ? step_by_lanes<float>(*a, s) : a->dtype == MB_F16 ? step_by_lanes<f16>(*a, s) : step_by_lanes<bf16>(*a, s);
}

}  // namespace ssm
}  // namespace mb

extern "C" size_t mb_selective_scan_workspace_bytes(const mb_selective_scan_args* a) {
  using namespace mb::ssm;
  if (check_scan("selective_scan_workspace_bytes", a, false) <= 0 || a->t == 0) return 0;  // mb_selective_scan says what is wrong
  Split sp;
  return split_layout(*a, nullptr, &sp);
}
extern "C" int mb_selective_scan(const mb_selective_scan_args* a, void* d_workspace, size_t workspace_bytes, mb_stream_t stream) {
  return mb::ssm::run_scan(a, d_workspace, workspace_bytes, (hipStream_t)stream);
}
extern "C" int mb_selective_scan_step(const mb_selective_scan_args* a, mb_stream_t stream) { return mb::ssm::run_step(a, (hipStream_t)stream); }
