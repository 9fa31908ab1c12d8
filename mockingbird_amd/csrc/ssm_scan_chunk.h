// The selective scan of prompts, a chunk of L rows at a time on the matrix pipe.  With a_t = d_t A and s(t) = a_1 + .. + a_t inside a chunk
//   y_t  = sum_{s <= t} (C_t . B_s) exp(s(t) - s(s)) d_s x_s + D x_t  +  exp(s(t)) (C_t . h)        h: the state in front of the chunk
//   h   <- exp(s(L)) h + sum_s exp(s(L) - s(s)) d_s x_s B_s^T
// i.e. four products per chunk and head: G = C B^T (shared by the heads of a group), M x, C h, and x^T B.
//
// A workgroup takes HB heads of one group and 64 of their columns (two waves per head, 32 columns each) and walks along time; h stays
// in the accumulators (fp32) of those waves for the whole walk and never visits LDS or memory between chunks.  Every product is written
// so that one factor is already in the register layout the matrix instruction wants: the accumulator layout of 16x16x32 products (column = lane
// & 15, rows 4 (lane >> 4) + i) of two stacked tiles IS an operand whose inner index runs 4 g + i, 16 + 4 g + i, so G^T feeds M x and
// h feeds C h directly, provided the other operand is read in the same order -- C as two 8-byte LDS reads, x^T and B^T as two
// transposing reads.
//
// Precision.  Every sum, the state and all exponents are fp32 (prefix sums over a chunk: fp64, so that differences of far rows keep
// their bits).  Operands are bf16 planes: a raw value is exact in 1 (bf16), 2 (fp16) or 3 (fp32) planes; computed operands are split as
// well -- M and h into two planes (2^-17 relative; three for fp32 calls) since y is rounded to 2^-9 or 2^-12 behind them, c_s x_s of the
// state into three, because the state is an fp32 result.  Products of planes below the last kept one are left out.
#pragma once
#include <atomic>
#include "ssm.h"

namespace mb {
namespace ssm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// exp and the step sizes are the library's fp32 functions: a decay error of one step is taken to the power of the sequence's length
__device__ __forceinline__ float step_raw(const mb_selective_scan_args& a, long long at) {
  return a.dt_dtype == MB_F32 ? ((const float*)a.d_dt)[at] : a.dt_dtype == MB_F16 ? to_f32(((const f16*)a.d_dt)[at]) : to_f32(((const bf16*)a.d_dt)[at]);
}
__device__ __forceinline__ float step_of(const mb_selective_scan_args& a, float d, int head) {
  if (a.d_dt_bias) d += a.d_dt_bias[head];
  if (a.dt_softplus) d = softplus(d);
  return d < a.dt_min ? a.dt_min : d > a.dt_max ? a.dt_max : d;  // NaN stays NaN
}
__device__ __forceinline__ float step_size(const mb_selective_scan_args& a, long long at, int head) { return step_of(a, step_raw(a, at), head); }

__device__ __forceinline__ float bf16_bits(unsigned short v) { return __uint_as_float((unsigned)v << 16); }

// Planes of 8 values: each the rounded remainder of those before it (Q planes carry 8 Q bits and a sign, the last one rounds).
// Two values at a time: one packed conversion, and their fp32 value back from its halves.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
template <int Q> __device__ __forceinline__ void split(const float (&v)[8], bf16x8 (&out)[Q]) {
  u32x4 w[Q];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const unsigned pair = pack_bf16(a, b);
      w[q][i] = pair;
      a -= __uint_as_float(pair << 16);
      b -= __uint_as_float(pair & 0xffff0000u);
    }
  }
#pragma unroll
  for (int q = 0; q < Q; ++q) out[q] = __builtin_bit_cast(bf16x8, w[q]);
}
// value i of 8 (by its 32-bit word)
__device__ __forceinline__ float value_of(const bf16x8& v, int i) {
  const u32x4 w = __builtin_bit_cast(u32x4, v);
  return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
}
// a NaN or infinity among 8 values
__device__ __forceinline__ bool not_finite(const bf16x8& v) {
  const u32x4 w = __builtin_bit_cast(u32x4, v);
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  return any;
}

// acc += a b over the plane pairs whose product is above 2^-8(K): K planes of the result are kept
template <int QA, int QB, int K>
__device__ __forceinline__ f32x4 mma(const bf16x8 (&a)[QA], const bf16x8 (&b)[QB], f32x4 acc) {
#pragma unroll
  for (int i = QA - 1; i >= 0; --i)
#pragma unroll
    for (int j = QB - 1; j >= 0; --j)
      if (i + j < K) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], acc, 0, 0, 0);
  return acc;
}

template <typename T, int NP> struct ScanShape {
  static constexpr int R = sizeof(T) == 4 ? 3 : std::is_same<T, f16>::value ? 2 : 1;  // raw planes
  static constexpr int Q = R == 3 ? 3 : 2;                                             // planes of M and h
  static constexpr int L = R == 1 && NP <= 128 ? 64 : 32;  // rows of a chunk: 64 where LDS and registers hold them
  static constexpr int HB = R == 3 && NP == 256 ? 2 : 4;   // heads of a workgroup
  static constexpr int PB = 64;                            // columns of a workgroup
  static constexpr int THREADS = HB * 128;
  static constexpr int TT = L / 16;                        // row tiles
  static constexpr int NT = NP / 16;                       // state tiles
  // LDS rows are 32 bytes longer than their data: 16 rows of 32 bytes (a wave's 8-byte and transposing reads) meet every bank twice
  static constexpr int NS = NP + 16, XS = PB + 16;         // row strides in halves
  static constexpr int GT = TT * (TT + 1) / 2;             // causal tiles of G
  struct alignas(16) Head { float u[L], w[L], pre[L], cs[L], hi[L], lo[L], d[L], f[TT][TT], total; };
  struct Lds {
    unsigned short b[R][L][NS], c[R][L][NS], x[HB][R][L][XS];
    f32x4 g[GT][64];
    Head head[HB];
  };
};

// Waves of a workgroup meet; LDS written before is visible behind it.  Loads from global memory stay in flight.
__device__ __forceinline__ void meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// 8 rows t (or s) of one column as an operand: rows t0 + 4 g + i and t0 + 16 + 4 g + i, column c0 + (lane & 15) of a row-major tile.
// Each group of 16 lanes hands in the 16 quads of its 4 rows and gets them back transposed.
template <int STRIDE> __device__ __forceinline__ bf16x8 read_transposed(const unsigned short (*m)[STRIDE], int t0, int c0, int lane) {
  typedef __attribute__((address_space(3))) s16x4 lds4;
  const int g = lane >> 4, i = lane & 15;
  const unsigned short* p = &m[t0 + 4 * g + (i >> 2)][c0 + 4 * (i & 3)];
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 16 * STRIDE));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(bf16x8, v);
}
// Row r of a row-major tile: columns c0 + 4 g + i and c0 + 16 + 4 g + i.
template <int STRIDE> __device__ __forceinline__ bf16x8 read_row(const unsigned short (*m)[STRIDE], int r, int c0, int g) {
  const bf16x4 lo = *(const bf16x4*)&m[r][c0 + 4 * g], hi = *(const bf16x4*)&m[r][c0 + 16 + 4 * g];
  return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// Raw values on their way to LDS: COUNT vectors of V per thread, requested a chunk ahead.  COLS (a power of two) values per row.
template <typename T, int V, int ROWS, int COLS, int THREADS> struct Stage {
  static constexpr int PER_ROW = COLS / V, TOTAL = ROWS * PER_ROW, COUNT = (TOTAL + THREADS - 1) / THREADS;
  Vec<T, V> v[COUNT];
  // col(c, n) -> offset of column c from the row, n = how many columns the tensor has from there on; rows from `rows` on are zero
  template <typename F> __device__ __forceinline__ void request(const T* base, long long rstride, int rows, F col) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const int at = (int)threadIdx.x + i * THREADS, r = at / PER_ROW, c = at % PER_ROW * V;
      int n = 0;
      const int off = col(c, n);
      v[i] = load_some<T, V>(base + r * rstride + off, r < rows ? n : 0);
    }
  }
  // put(plane, row, column, V halves)
  template <int R, typename F> __device__ __forceinline__ void lay(F put) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const int at = (int)threadIdx.x + i * THREADS, r = at / PER_ROW, c = at % PER_ROW * V;
      if (TOTAL % THREADS != 0 && r >= ROWS) continue;
      if constexpr (R == 1) {
        put(0, r, c, __builtin_bit_cast(Vec<unsigned short, V>, v[i]));
      } else {
        float f[V];
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = to_f32(v[i].v[k]);
#pragma unroll
        for (int q = 0; q < R; ++q) {
          Vec<unsigned short, V> h;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            h.v[k] = __builtin_bit_cast(unsigned short, (__bf16)f[k]);
            // an fp32 value above bf16's range is cut instead of rounded to infinity
            if (R == 3 && q == 0 && (h.v[k] & 0x7fff) == 0x7f80) h.v[k] = (unsigned short)(__float_as_uint(f[k]) >> 16);
            f[k] -= bf16_bits(h.v[k]);
          }
          put(q, r, c, h);
        }
      }
    }
  }
};

// Workspace of a call that is split along time: per tile of `seg` rows and head the state it adds, then the state in front of it, and its decay.
struct Split {
  float* state;  // [tiles][heads][head_dim][d_state]
  float* decay;  // [tiles][heads]
  int seg;       // rows of a tile, a multiple of L; 0: not split
};

// STATES: first pass of a split call, the state every tile adds to a zero state.  Otherwise y (and the final states).
template <typename T, int NP, bool STATES>
__global__ __launch_bounds__((ScanShape<T, NP>::THREADS)) void selective_scan_chunk_kernel(const mb_selective_scan_args a, const Split sp) {
  typedef ScanShape<T, NP> S;
  constexpr int V = 16 / sizeof(T), R = S::R, Q = S::Q, L = S::L, HB = S::HB, TT = S::TT, NT = S::NT, PB = S::PB, THREADS = S::THREADS;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  typename S::Lds& m = *(typename S::Lds*)lds_raw;

  const int per_group = a.heads / a.groups, hblocks = (per_group + HB - 1) / HB, pblocks = (a.head_dim + PB - 1) / PB;
  const int units = a.groups * hblocks * pblocks;
  const unsigned tile = blockIdx.x / units;
  int u = (int)(blockIdx.x - tile * units);
  const int pb = u % pblocks;
  u /= pblocks;
  const int hb = u % hblocks, group = u / hblocks;
  const int head0 = group * per_group + hb * HB, live = min(HB, per_group - hb * HB);
  const int p0 = pb * PB;

  const Rows rows = {a.d_cu_seqlens, a.d_valid, a.batch, a.t};
  const int seg = sp.seg ? sp.seg : max(a.t, 1);
  const Item it = item_of(rows, tile, seg);
  const int parts = max(1, (it.len + seg - 1) / seg);
  if (it.part < 0 || it.part >= parts || (STATES && it.part == parts - 1)) return;  // nobody asks what the last part adds
  int slot = -1;
  if (a.d_state) {
    slot = slot_of(a.d_slots, it.b, a.n_slots);
    if (slot < 0) return;
  }
  const int t0 = it.part * seg, t1 = min(it.len, t0 + seg);
  const long long pad = a.d_cu_seqlens ? 0 : it.b;
  const T* xg = (const T*)a.d_x + pad * a.x_bstride + it.row * a.x_rstride + (long long)head0 * a.head_dim + p0;
  const T* bg = (const T*)a.d_b + pad * a.b_bstride + it.row * a.b_rstride + (long long)group * a.d_state_dim;
  const T* cg = (const T*)a.d_c + pad * a.c_bstride + it.row * a.c_rstride + (long long)group * a.d_state_dim;
  T* yg = (T*)a.d_y + pad * a.y_bstride + it.row * a.y_rstride + (long long)head0 * a.head_dim + p0;
  const long long dtg = pad * a.dt_bstride + it.row * a.dt_rstride;

  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63, g = lane >> 4, li = lane & 15;
  const int hh = wave % HB, half = wave / HB, head = head0 + min(hh, live - 1);
  const bool mine = hh < live;
  const int pw = half * 32;  // this wave's columns p0 + pw .. + 31

  f32x4 h[2][NT];  // [column tile][state tile]: h[n = 16 nt + 4 g + i][p = p0 + pw + 16 pt + li]
  float* st = nullptr;
  const long long head_state = (long long)a.head_dim * a.d_state_dim;
  if (a.d_state && !sp.seg) st = a.d_state + slot * a.state_stride + head * head_state;
  const float* from = sp.seg ? sp.state + ((long long)tile * a.heads + head) * head_state : st;
  const bool keep = !STATES && (sp.seg ? true : st && (!a.d_has_state || a.d_has_state[it.b]));
#pragma unroll
  for (int pt = 0; pt < 2; ++pt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int p = p0 + pw + 16 * pt + li, n = 16 * nt + 4 * g;
      const int left = keep && mine && p < a.head_dim ? a.d_state_dim - n : 0;
      h[pt][nt] = __builtin_bit_cast(f32x4, load_some<float, 4>(from + (long long)p * a.d_state_dim + n, left));
    }

  Stage<T, V, L, NP, THREADS> sb, sc;
  Stage<T, V, L, HB * PB, THREADS> sx;
  float draw = 0.f;
  auto request = [&](int t) {
    const int n = t1 - t;
    auto col_n = [&](int c, int& left) {
      left = a.d_state_dim - c;
      return c;
    };
    sb.request(bg + t * a.b_rstride, a.b_rstride, n, col_n);
    if (!STATES) sc.request(cg + t * a.c_rstride, a.c_rstride, n, col_n);
    sx.request(xg + t * a.x_rstride, a.x_rstride, n, [&](int c, int& left) {
      const int i = c / PB, p = c % PB;
      left = i < live ? a.head_dim - p0 - p : 0;
      return i * a.head_dim + p;
    });
    if (half == 0 && mine && lane < L && lane < n) draw = step_raw(a, dtg + (t + lane) * a.dt_rstride + head);
  };
  const float A = a.d_a[head], skip = a.d_d ? a.d_d[head] : 0.f;
  // everything of a chunk that depends on the step sizes alone, one lane per row
  double walked = 0.0;  // sum of a over the tile so far: its decay
  auto scalars = [&](int t) {
    if (half != 0 || !mine) return;
    const bool in = lane < L && t + lane < t1;
    const float d = in ? step_of(a, draw, head) : 0.f;
    double s = in ? (double)d * (double)A : 0.0;
#pragma unroll
    for (int o = 1; o < L; o *= 2) {
      const double up = __shfl_up(s, o, 64);
      if (lane >= o) s += up;
    }
    const double before = __shfl(s, (lane & ~15) - 1, 64), tile_end = __shfl(s, lane | 15, 64), end = __shfl(s, L - 1, 64);
    const double start = lane < 16 ? 0.0 : before;
    typename S::Head& o = m.head[hh];
    if (lane < L) {
      const double local = s - start;
      o.u[lane] = expf((float)local);
      o.w[lane] = expf((float)(tile_end - s)) * d;
      o.pre[lane] = expf((float)s);
      o.cs[lane] = expf((float)(end - s)) * d;
      const float hi = (float)s;
      o.hi[lane] = hi;
      o.lo[lane] = (float)(s - (double)hi);
      o.d[lane] = d;
    }
    // f[i][j]: from the end of tile i to the start of tile j
    const int i = lane / TT % TT, j = lane % TT;
    const double fi = __shfl(s, 16 * i + 15, 64), fj = __shfl(s, j ? 16 * j - 1 : 0, 64);
    if (lane < TT * TT && i < j) o.f[i][j] = expf((float)(fj - fi));
    if (lane == 0) o.total = expf((float)end);
    walked += end;
  };
  auto lay = [&]() {
    sb.template lay<R>([&](int q, int r, int c, const Vec<unsigned short, V>& v) { store_vec<unsigned short, V>(&m.b[q][r][c], v); });
    if (!STATES) sc.template lay<R>([&](int q, int r, int c, const Vec<unsigned short, V>& v) { store_vec<unsigned short, V>(&m.c[q][r][c], v); });
    sx.template lay<R>([&](int q, int r, int c, const Vec<unsigned short, V>& v) { store_vec<unsigned short, V>(&m.x[c / PB][q][r][c % PB], v); });
  };

  if (t0 < t1) request(t0);
  for (int t = t0; t < t1; t += L) {
    lay();
    scalars(t);
    meet();
    if (t + L < t1) request(t + L);

    f32x4 acc[TT][2];
    const typename S::Head& hd = m.head[hh];
    if (!STATES) {
      // G^T, tiles (s tile i <= t tile j), dealt to the waves
      for (int k = wave; k < S::GT; k += THREADS / 64) {
        int j = 0;
        while ((j + 1) * (j + 2) / 2 <= k) ++j;
        const int i = k - j * (j + 1) / 2;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NP; n += 32) {
          bf16x8 fa[R], fb[R];
#pragma unroll
          for (int q = 0; q < R; ++q) {
            fa[q] = read_row<S::NS>(m.b[q], 16 * i + li, n, g);
            fb[q] = read_row<S::NS>(m.c[q], 16 * j + li, n, g);
          }
          s = mma<R, R, R>(fa, fb, s);
        }
        m.g[k][lane] = s;
      }
      // C h, scaled to each row's distance from the state
      if (mine) {
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[j][0] = acc[j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          bf16x8 fh[2][Q];
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
            const f32x4 lo = h[pt][n], hi = h[pt][n + 1];
            const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            split<Q>(v, fh[pt]);
          }
#pragma unroll
          for (int j = 0; j < TT; ++j) {
            bf16x8 fc[R];
#pragma unroll
            for (int q = 0; q < R; ++q) fc[q] = read_row<S::NS>(m.c[q], 16 * j + li, 16 * n, g);
#pragma unroll
            for (int pt = 0; pt < 2; ++pt) acc[j][pt] = mma<Q, R, Q>(fh[pt], fc, acc[j][pt]);
          }
        }
#pragma unroll
        for (int j = 0; j < TT; ++j) {
          const float pre = hd.pre[16 * j + li];
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) acc[j][pt] *= pre;
        }
      }
      meet();
    }
    if (mine) {
      bf16x8 fx[2][L / 32][R];
      bool any = false;
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int k = 0; k < L / 32; ++k)
#pragma unroll
          for (int q = 0; q < R; ++q) {
            fx[pt][k][q] = read_transposed<S::XS>(m.x[hh][q], 32 * k, pw + 16 * pt, lane);
            any |= not_finite(fx[pt][k][q]);
          }
      // h <- total h + B^T (c x)
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) h[pt][nt] *= hd.total;
#pragma unroll
      for (int k = 0; k < L / 32; ++k) {
        const f32x4 c0 = *(const f32x4*)&hd.cs[32 * k + 4 * g], c1 = *(const f32x4*)&hd.cs[32 * k + 16 + 4 * g];
        bf16x8 fs[2][3];
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float xv = 0.f;
#pragma unroll
            for (int q = R - 1; q >= 0; --q) xv += value_of(fx[pt][k][q], i);
            v[i] = (i < 4 ? c0[i & 3] : c1[i & 3]) * xv;
          }
          split<3>(v, fs[pt]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          bf16x8 fb[R];
#pragma unroll
          for (int q = 0; q < R; ++q) fb[q] = read_transposed<S::NS>(m.b[q], 32 * k, 16 * nt, lane);
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) h[pt][nt] = mma<R, 3, 3>(fb, fs[pt], h[pt][nt]);
        }
      }
      if (!STATES) {
        // 0 * NaN in the half of M that is zero would reach rows in front of the NaN: such elements are taken out of the product, and
        // their column's rows from there on are set to NaN below
        int bad[2] = {L, L};  // first such row of this lane's columns
        const bool poisoned = __any(any);
        if (poisoned) {
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
#pragma unroll
            for (int k = 0; k < L / 32; ++k)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                bool b = false;
#pragma unroll
                for (int q = 0; q < R; ++q) b |= !(fabsf(value_of(fx[pt][k][q], i)) <= 3.4e38f);
                if (b) {
                  bad[pt] = min(bad[pt], 32 * k + (i < 4 ? 4 * g + i : 12 + 4 * g + i));
#pragma unroll
                  for (int q = 0; q < R; ++q) fx[pt][k][q][i] = (__bf16)0.f;
                }
              }
            bad[pt] = min(bad[pt], __shfl_xor(bad[pt], 16, 64));
            bad[pt] = min(bad[pt], __shfl_xor(bad[pt], 32, 64));
          }
        }
#pragma unroll
        for (int j = 0; j < TT; ++j) {
          const float u = hd.u[16 * j + li], thi = hd.hi[16 * j + li], tlo = hd.lo[16 * j + li];
#pragma unroll
          for (int k = 0; k <= j / 2; ++k) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int i = 2 * k + e;
              if (i > j) {
#pragma unroll
                for (int r = 0; r < 4; ++r) v[4 * e + r] = 0.f;
                continue;
              }
              const f32x4 gt = m.g[j * (j + 1) / 2 + i][lane];
              if (i < j) {
                const f32x4 w = *(const f32x4*)&hd.w[16 * i + 4 * g];
                const float uf = u * hd.f[i][j];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[4 * e + r] = gt[r] * (uf * w[r]);
              } else {
                const f32x4 shi = *(const f32x4*)&hd.hi[16 * i + 4 * g], slo = *(const f32x4*)&hd.lo[16 * i + 4 * g];
                const f32x4 d = *(const f32x4*)&hd.d[16 * i + 4 * g];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const int s = 4 * g + r;
                  // the two differences of hi + lo parts are exact or as good as the exponent's own rounding
                  float c = gt[r] * (expf((thi - shi[r]) + (tlo - slo[r])) * d[r]);
                  if (s == li) c = fmaf(gt[r], d[r], skip);
                  v[4 * e + r] = s <= li ? c : 0.f;
                }
              }
            }
            bf16x8 fm[Q];
            split<Q>(v, fm);
#pragma unroll
            for (int pt = 0; pt < 2; ++pt) acc[j][pt] = mma<R, Q, Q>(fx[pt][k], fm, acc[j][pt]);
          }
          // y^T tile: row p = 4 g + i, column t = li
          const int row = t + 16 * j + li;
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
            if (poisoned) {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (16 * j + li >= __shfl(bad[pt], 4 * g + r, 64)) acc[j][pt][r] = __builtin_nanf("");
            }
            const int p = p0 + pw + 16 * pt + 4 * g;
            if (row < t1) {
              T* dst = yg + row * a.y_rstride + (long long)hh * a.head_dim + pw + 16 * pt + 4 * g;
              Vec<T, 4> o;
#pragma unroll
              for (int r = 0; r < 4; ++r) o.v[r] = from_f32<T>(acc[j][pt][r]);
              store_some<T, 4>(dst, o, a.head_dim - p);
            }
          }
        }
      }
    }
    meet();
  }

  if (STATES) {
    if (half == 0 && mine && lane == 0) sp.decay[(long long)tile * a.heads + head] = expf((float)walked);
  } else if (!a.d_state || it.part != parts - 1) {
    return;
  }
  if (!mine) return;
  float* to = STATES ? sp.state + ((long long)tile * a.heads + head) * head_state : a.d_state + slot * a.state_stride + head * head_state;
#pragma unroll
  for (int pt = 0; pt < 2; ++pt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int p = p0 + pw + 16 * pt + li, n = 16 * nt + 4 * g;
      if (p < a.head_dim) store_some<float, 4>(to + (long long)p * a.d_state_dim + n, __builtin_bit_cast(Vec<float, 4>, h[pt][nt]), a.d_state_dim - n);
    }
}

template <typename T, int NP, bool STATES> int launch_chunk(const mb_selective_scan_args& a, const Split& sp, hipStream_t s) {
  typedef ScanShape<T, NP> S;
  static_assert(sizeof(typename S::Lds) <= 160 * 1024, "a chunk has to fit LDS");
  static std::atomic<unsigned long long> attr_done{0};  // per device: the attribute belongs to the function on the current device
  int dev = 0;
  MB_HIP(hipGetDevice(&dev));
  const unsigned long long bit = dev >= 0 && dev < 64 ? 1ull << dev : 0ull;
  if (!bit || !(attr_done.load(std::memory_order_acquire) & bit)) {
    MB_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&selective_scan_chunk_kernel<T, NP, STATES>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    attr_done.fetch_or(bit, std::memory_order_release);
  }
  const Rows rows = {a.d_cu_seqlens, a.d_valid, a.batch, a.t};
  const int per_group = a.heads / a.groups;
  const long long units = (long long)a.groups * cdiv(per_group, S::HB) * cdiv(a.head_dim, S::PB);
  const long long grid = tiles_of(rows, sp.seg ? sp.seg : (a.t > 1 ? a.t : 1)) * units;
  MB_REQUIRE(grid < (1ll << 31), "selective_scan: %d items of %d heads are too many for one launch", a.batch, a.heads);
  hipLaunchKernelGGL((selective_scan_chunk_kernel<T, NP, STATES>), dim3((unsigned)grid), dim3(S::THREADS), sizeof(typename S::Lds), s, a, sp);
  MB_HIP(hipGetLastError());
  return MB_OK;
}

template <typename T> int chunk_launch(const mb_selective_scan_args& a, const Split& sp, bool states, hipStream_t s) {
  if (a.d_state_dim <= 64) return states ? launch_chunk<T, 64, true>(a, sp, s) : launch_chunk<T, 64, false>(a, sp, s);
  if (a.d_state_dim <= 128) return states ? launch_chunk<T, 128, true>(a, sp, s) : launch_chunk<T, 128, false>(a, sp, s);
  return states ? launch_chunk<T, 256, true>(a, sp, s) : launch_chunk<T, 256, false>(a, sp, s);
}

// the kernels of one type each, in ssm_scan_{f32,f16,bf16}.hip
int scan_chunks_f32(const mb_selective_scan_args& a, const Split& sp, bool states, hipStream_t s);
int scan_chunks_f16(const mb_selective_scan_args& a, const Split& sp, bool states, hipStream_t s);
int scan_chunks_bf16(const mb_selective_scan_args& a, const Split& sp, bool states, hipStream_t s);

}  // namespace ssm
}  // namespace mb
