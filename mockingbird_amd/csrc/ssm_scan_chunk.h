// The selective scan of prompts, a chunk of L rows at a time on the matrix pipe.  With a_t = d_t A and s(t) = a_1 + .. + a_t inside a chunk
//   y_t  = sum_{s <= t} (C_t . B_s) exp(s(t) - s(s)) d_s x_s + D x_t  +  exp(s(t)) (C_t . h)        h: the state in front of the chunk
//   h   <- exp(s(L)) h + sum_s exp(s(L) - s(s)) d_s x_s B_s^T
// i.e. four products per chunk and head: G = C B^T (shared by the heads of a group), M x, C h, and x^T B.
//
// A workgroup takes two heads of one group and 64 of their columns (four waves per head, 16 columns each) and walks along time; h stays
// in the accumulators (fp32) of those waves for the whole walk and never visits LDS or memory between chunks.  Every product is written
// so that one factor is already in the register layout the matrix instruction wants: in the accumulators of two stacked 16x16x32 tiles a
// lane holds rows 4 g + i of both (g = lane >> 4) of column lane & 15, which is an operand whose inner index is dealt out as those rows.
// So G^T tiles become M^T operands and h tiles operands of C h without moving between lanes, provided the other operand is read in the same
// order: x^T by transposing reads of rows 4 g + i and 16 + 4 g + i; for C h the state's rows are numbered so that the order is C's own
// (tile 2 q holds columns 32 q + 8 g + i, tile 2 q + 1 those 4 further on).
//
// What bounds it: per wave and chunk 97 matrix instructions and about 580 vector ones, most of which split h, M and c x into planes, take 25 %
// and 38 % of the time of their pipes and overlap by half at best; the rest is the order of a chunk -- step sizes, G, M, M x, three meetings of
// the waves (41 % of their time is waiting; 60 vector instructions fewer gave 1 %).  Hence: M is formed once per head and goes through LDS; two
// workgroups of 8 waves fit a CU (78 KB of LDS, 128 registers; nothing spilled at 128 states -- a reload waits for the loads in flight in
// front of it -- while bf16 at 256 states spills 15 registers, and sizes that are not whole tiles 6 at 128 states and 86 at 256), so that one's
// products run while the other waits; the terms of the step sizes are a chunk ahead; the conversion of the next operand stands between the
// products of this one.  Four waves of 32 columns read LDS half as often and are no faster (8192 rows, 64 heads of 64 x 128: 149 and 146 us),
// one workgroup of four heads neither, nor the second pass adding up the tiles in front of its own instead of a join (156 and 137 us).
// Measured, 8192 rows x 64 heads of 64 columns, 128 states, bf16: 86 us this pass (at best 78), 43 (40) the states' pass, 14 the join between
// them, of 28 us that its bytes take at a large copy's rate.  Planes less would save 9 us (h and M in one) and 10 us (c x in two) of it.
// Sizes that are not whole tiles load and lay down in one go, nothing ahead: 48 heads of 96 x 100 take 219 us where 64 of 64 x 128 take 137;
// narrow heads and small states are computed as 64 columns and states: 64 heads of 32 x 16 take 98 us.
//
// Precision.  Every sum, the state and all exponents are fp32 (prefix sums over a chunk: fp64, so that differences of far rows keep
// their bits).  Operands are bf16 planes: a raw value is exact in 1 (bf16), 2 (fp16) or 3 (fp32) planes; computed operands are split as
// well -- M and h into two planes (2^-17 relative; three for fp32 calls) since y is rounded to 2^-9 or 2^-12 behind them, c_s x_s of the
// state into three, because the state is an fp32 result.  Products of planes below the last kept one are left out: up to 2^-18 of each term
// of G, C h and M x in fp16 calls, 2^-25 in fp32 ones.  So a 16-bit y is a plain fp32 evaluation's up to single last places (in 0.1 % of a
// bf16 result, 1 % of an fp16 one) unless its terms cancel to less than about 2^-8 (bf16) or 2^-5 (fp16) of their size, and the state is an fp32 evaluation's.
#pragma once
#include <atomic>
#include "ssm.h"

namespace mb {
namespace ssm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Step sizes and decays keep fp32's full accuracy whatever the activations' type: a decay's error is taken to the power of the rows it spans.
__device__ __forceinline__ float step_raw(const mb_selective_scan_args& a, long long at) {
  return a.dt_dtype == MB_F32 ? ((const float*)a.d_dt)[at] : a.dt_dtype == MB_F16 ? to_f32(((const f16*)a.d_dt)[at]) : to_f32(((const bf16*)a.d_dt)[at]);
}
__device__ __forceinline__ float step_of(const mb_selective_scan_args& a, float d, float bias) {
  d += bias;
  if (a.dt_softplus) d = softplus(d);
  return d < a.dt_min ? a.dt_min : d > a.dt_max ? a.dt_max : d;  // NaN stays NaN
}
__device__ __forceinline__ float step_size(const mb_selective_scan_args& a, long long at, int head) {
  return step_of(a, step_raw(a, at), a.d_dt_bias ? a.d_dt_bias[head] : 0.f);
}

__device__ __forceinline__ float bf16_bits(unsigned short v) { return __uint_as_float((unsigned)v << 16); }

// Schedule of a region: DS_FIRST LDS reads, then MFMAS matrix instructions with up to VALU vector instructions behind each and the rest of
// the DS LDS reads spread over them.  Without it the conversions of the next operands come in one block, and neither pipe runs beside the other.
template <int MFMAS, int VALU, int DS, int DS_FIRST> __device__ __forceinline__ void behind_each() {
  __builtin_amdgcn_sched_group_barrier(0x100, DS_FIRST, 0);
#pragma unroll
  for (int i = 0; i < MFMAS; ++i) {
    constexpr int REST = DS - DS_FIRST;
    if ((i + 1) * REST / MFMAS - i * REST / MFMAS == 1) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    if ((i + 1) * REST / MFMAS - i * REST / MFMAS == 2) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}
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

template <typename T, int NP, bool STATES> struct ScanShape {
  static constexpr int R = sizeof(T) == 4 ? 3 : std::is_same<T, f16>::value ? 2 : 1;  // raw planes
  static constexpr int Q = R == 3 ? 3 : 2;                                             // planes of M and h
  static constexpr int L = R == 1 && NP <= 128 ? 64 : 32;  // rows of a chunk: 64 where two workgroups' LDS and registers hold them
  static constexpr int HB = 2;                             // heads of a workgroup
  static constexpr int PB = 64;                            // columns of a workgroup
  static constexpr int WPH = PB / 16;                      // waves per head: 16 columns each
  static constexpr int CH_PAIRS = R == 1 ? 2 : R == 2 ? 3 : 6, ST_PAIRS = R == 1 ? 3 : R == 2 ? 5 : 6;  // products per operand pair
  static constexpr int THREADS = HB * WPH * 64;
  static constexpr int TT = L / 16;                        // row tiles
  static constexpr int NT = NP / 16;                       // state tiles
  // LDS rows of B and C are 32 bytes longer than their data: 8 rows of one 16-byte unit lie in different banks.  x has no room for that (two
  // workgroups would not fit): its 32-byte pieces change places with the row, so that 4 rows of one piece do.
  static constexpr int NS = NP + 16;                       // row stride in halves
  static __device__ __forceinline__ unsigned x_col(unsigned r, unsigned c) { return c ^ 16 * (r >> 1 & 1); }
  static constexpr int GT = TT * (TT + 1) / 2;             // causal tiles of G
  struct alignas(16) Head { float u[L], w[L], hi[L], lo[L], d[L], f[TT][TT], front[TT], back[TT], total; };
  // Step-size terms of HEADS chunks.  The states' pass, which needs no C and no M, has room for 8: every wave of a head does one of the next
  // four chunks at a time.  The other pass keeps this chunk's and the next one's, which one wave of each head does.
  static constexpr int HEADS = STATES ? 2 * WPH : 2;
  struct LdsY { unsigned short c[R][L][NS]; bf16x4 m[HB][GT * Q * 64]; };
  // Two s tiles of M^T next to each other are one operand of 32 rows (16 bytes a lane); the diagonal tiles of even rows of tiles have no
  // partner and come first.  -> index of tile (i, j), plane q, this lane
  static __device__ __forceinline__ int m_at(int i, int j, int q, int lane) {
    if (i == j && i % 2 == 0) return (j / 2 * Q + q) * 64 + lane;
    return TT / 2 * Q * 64 + 2 * ((pairs_before(j) + i / 2) * Q + q) * 64 + 2 * lane + i % 2;
  }
  static __device__ __forceinline__ int pairs_before(int j) { return (j / 2) * (j / 2) + (j % 2) * (j / 2); }  // in rows of tiles 0 .. j - 1
  struct LdsStates { double walked[HB][WPH]; };
  struct Lds : std::conditional<STATES, LdsStates, LdsY>::type {
    unsigned short b[R][L][NS], x[HB][R][L][PB];
    Head head[HEADS][HB];
    int odd[HB][WPH];  // step sizes that the products cannot do
  };
  static constexpr int WAVES = (sizeof(Lds) <= 80 * 1024 ? 2 : 1) * THREADS / 256;  // per SIMD, of the workgroups that share a CU
};

// Waves of a workgroup meet; LDS written before is visible behind it.  Loads from global memory stay in flight.
__device__ __forceinline__ void meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// 8 rows of one column as an operand, out of LDS: each group of 16 lanes hands in the quads (4 columns) of its 4 rows and gets the 16
// columns back transposed.  lo: this lane's quad in rows 4 g + i, hi: in rows 16 + 4 g + i.
__device__ __forceinline__ bf16x8 read_transposed(const unsigned short* lo, const unsigned short* hi) {
  typedef __attribute__((address_space(3))) s16x4 lds4;
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)lo), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)hi);
  const s16x8 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  return __builtin_bit_cast(bf16x8, v);
}
template <int V> __device__ __forceinline__ void store_lds(unsigned short* p, const Vec<unsigned short, V>& v) {
  typedef unsigned short vt __attribute__((ext_vector_type(V)));
  *(vt*)p = __builtin_bit_cast(vt, v);  // aligned: rows of 16-byte multiples, columns of V
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
  // The same where every column exists: through a buffer descriptor that ends behind row `rows` - 1, whose range check supplies the zeros.
  // One address register for all; the thread's further vectors are a fixed number of rows on.
  static __device__ __forceinline__ unsigned offset(unsigned tid, int rstride) {
    return (tid / PER_ROW * (unsigned)rstride + tid % PER_ROW * V) * (unsigned)sizeof(T);
  }
  __device__ __forceinline__ void request(const T* base, int rstride, int rows, unsigned off, int width) {
    // (31 bits hold it: the host looked)
    const __amdgpu_buffer_rsrc_t d = tm_rsrc(base, rows > 0 ? ((rows - 1) * rstride + width) * (int)sizeof(T) : 0);
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      v[i] = __builtin_bit_cast(Vec<T, V>, __builtin_amdgcn_raw_buffer_load_b128(d, off, i * (THREADS / PER_ROW) * rstride * (int)sizeof(T), 0));
  }
  // put(plane, row, column, V halves)
  template <int R, typename F> __device__ __forceinline__ void lay(unsigned tid, F put) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const unsigned at = tid + i * THREADS, r = at / PER_ROW, c = at % PER_ROW * V;
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

// Workspace of a call that is split along time: for every tile of `seg` rows that has one behind it, in the order of items and rows, and every
// head what it adds to the state, and its decay; the join puts the state in front of the next tile in the sum's place.  The state in front
// of an item's first tile is in the pool, where the last tile leaves the new one: split items have a copy.
struct Split {
  float* state;   // [fronts][heads][head_dim][d_state]
  float* initial; // [initials][heads][head_dim][d_state]
  float* decay;   // [fronts][heads]; -0: a row's own decay is zero, 0: only their product is
  int seg;        // rows of a tile, a multiple of L; 0: not split
  int fronts, initials;
};
// Where the copy of item b's state is; `before` tiles of earlier items have one behind them.  (-1, for lists of overlapping rows: there is none)
__device__ __forceinline__ int initial_at(const Split& sp, int batch, int b, int before) {
  if (batch <= sp.initials) return b;
  return (unsigned)before < (unsigned)sp.initials ? before : -1;
}

__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
// prefix sum over the 16 lanes of a row: shifts within the row bring in zeros
template <int N> __device__ __forceinline__ double row_shifted(double v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, 0x110 + N, 0xf, 0xf, true);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), 0x110 + N, 0xf, 0xf, true);
  return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double from_lane(double v, int lane) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)b, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(b >> 32), lane);
  return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}

// What a workgroup works on, from its number.
template <typename T> struct Work {
  const T *x, *b, *c;     // row 0 of the item: the first head's columns p0 .., the group's B and C
  T* y;                   // this wave's columns
  long long dt;
  float* pool;            // this wave's head: its state, null without a pool
  const float* from;      // and the state in front of the tile, if `carried`
  unsigned tile;
  int part, parts, t0, t1, p0, head0, live, head, columns;
  bool carried, none;     // none: nothing to do
};
template <typename T, int NP, bool STATES, bool WHOLE>
__device__ __forceinline__ Work<T> work_of(const mb_selective_scan_args& a, const Split& sp, unsigned block, int wave) {
  typedef ScanShape<T, NP, STATES> S;
  constexpr int HB = S::HB, PB = S::PB;
  Work<T> w;
  w.none = true;
  const int head_dim = a.head_dim, d_state = WHOLE ? NP : a.d_state_dim;
  const int per_group = a.heads / a.groups, hblocks = (per_group + HB - 1) / HB, pblocks = (head_dim + PB - 1) / PB;
  const int units = a.groups * hblocks * pblocks;
  w.tile = block / units;
  int unit = (int)(block - w.tile * units);
  w.p0 = unit % pblocks * PB;
  unit /= pblocks;
  const int hb = unit % hblocks, group = unit / hblocks;
  w.head0 = group * per_group + hb * HB, w.live = WHOLE ? HB : min(HB, per_group - hb * HB);

  const Rows rows = {a.d_cu_seqlens, a.d_valid, a.batch, a.t};
  const int seg = sp.seg ? sp.seg : max(a.t, 1);
  const Item it = item_of(rows, w.tile, seg, STATES);  // nobody asks what the last part adds
  w.part = it.part, w.parts = max(1, (it.len + seg - 1) / seg);
  if (it.part < 0 || it.part >= w.parts) return w;
  int slot = -1;
  if (a.d_state) {
    slot = slot_of(a.d_slots, it.b, a.n_slots);
    if (slot < 0) return w;
  }
  w.t0 = it.part * seg, w.t1 = min(it.len, w.t0 + seg);
  const long long pad = a.d_cu_seqlens ? 0 : it.b;
  w.x = (const T*)a.d_x + pad * a.x_bstride + it.row * a.x_rstride + (long long)w.head0 * head_dim + w.p0;
  w.b = (const T*)a.d_b + pad * a.b_bstride + it.row * a.b_rstride + (long long)group * d_state;
  w.c = (const T*)a.d_c + pad * a.c_bstride + it.row * a.c_rstride + (long long)group * d_state;
  w.dt = pad * a.dt_bstride + it.row * a.dt_rstride;
  w.head = w.head0 + min(wave % HB, w.live - 1);
  w.columns = wave / HB * 16;  // p0 + these ..
  w.y = (T*)a.d_y + pad * a.y_bstride + it.row * a.y_rstride + (long long)w.head * head_dim + w.p0 + w.columns;
  const long long head_state = (long long)head_dim * d_state;
  w.pool = a.d_state ? a.d_state + slot * a.state_stride + w.head * head_state : nullptr;
  w.from = w.pool;  // an item of one part is not split
  w.carried = !STATES && (it.part > 0 || (w.pool && (!a.d_has_state || a.d_has_state[it.b])));
  if (w.carried && w.parts > 1) {
    const int before = (int)w.tile - it.b;  // tiles in front of this one that have one behind them
    const int at = it.part ? before - 1 : initial_at(sp, a.batch, it.b, before);
    if (it.part ? (unsigned)at >= (unsigned)sp.fronts : at < 0) return w;  // (lists of overlapping rows; all waves)
    w.from = (it.part ? sp.state : sp.initial) + ((long long)at * a.heads + w.head) * head_state;
  }
  w.none = false;
  return w;
}
// h[2 q + e]: column p0 + columns + (lane & 15), state columns 32 q + 8 g + 4 e + i
template <typename T, int NP, bool WHOLE> __device__ __forceinline__ void start_of(const Work<T>& w, int head_dim, int d_state, bool mine, int lane, f32x4 (&h)[NP / 16]) {
#pragma unroll
  for (int nt = 0; nt < NP / 16; ++nt) {
    const int p = w.p0 + w.columns + (lane & 15), n = nt / 2 * 32 + 8 * (lane >> 4) + nt % 2 * 4;
    const int left = w.carried && mine && (WHOLE || p < head_dim) ? (WHOLE ? 4 : d_state - n) : 0;
    h[nt] = __builtin_bit_cast(f32x4, load_some<float, 4>(w.from + (long long)p * d_state + n, left));
  }
}

// The tile again, row by row, each wave its own columns: where infinities, NaN or growth beyond fp32 keep the products from giving what the
// recurrence gives.  (8192 rows, 64 heads of 64 x 128 bf16 with a NaN in every head: 1.9 ms instead of 0.13.)  It is called behind the
// products, so nothing it needs is kept through them: the arguments are read anew from the kernel's own.
template <typename T, int NP, bool STATES, bool WHOLE> __device__ __forceinline__ void walk_rows(f32x4 (&h)[NP / 16]) {
  struct Args {
    mb_selective_scan_args a;
    Split sp;
  };
  typedef __attribute__((address_space(4))) const Args Given;
  Given* given = (Given*)__builtin_amdgcn_kernarg_segment_ptr();
  unsigned block = blockIdx.x;
  asm volatile("" : "+s"(given), "+s"(block));
  Args args;
  __builtin_memcpy(&args, (const void*)given, sizeof(Args));
  const mb_selective_scan_args& a = args.a;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63, g = lane >> 4, li = lane & 15;
  const Work<T> w = work_of<T, NP, STATES, WHOLE>(a, args.sp, block, wave);
  const int d_state = WHOLE ? NP : a.d_state_dim, column = w.p0 + w.columns + li;
  const bool there = WHOLE || column < a.head_dim;
  start_of<T, NP, WHOLE>(w, a.head_dim, d_state, true, lane, h);
  const T* x = w.x + (w.head - w.head0) * a.head_dim + w.columns + li;
  const float A = a.d_a[w.head], skip = a.d_d ? a.d_d[w.head] : 0.f;
  __threadfence();  // the answers below go behind those of the products
  for (int t = w.t0; t < w.t1; ++t) {
    const float d = step_size(a, w.dt + t * a.dt_rstride + w.head, w.head), decay = expf(d * A);
    const float xv = there ? to_f32(x[t * a.x_rstride]) : 0.f, dx = d * xv;
    float y = 0.f;
    int fresh = lane;
    asm volatile("" : "+v"(fresh));  // (masks and addresses by column are not worth registers of the loop)
#pragma unroll
    for (int nt = 0; nt < NP / 16; ++nt) {
      const int n = nt / 2 * 32 + 8 * (fresh >> 4) + nt % 2 * 4;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = WHOLE ? n + r : min(n + r, d_state - 1);
        const float bv = to_f32(w.b[t * a.b_rstride + at]), cv = STATES ? 0.f : to_f32(w.c[t * a.c_rstride + at]);
        const float next = fmaf(h[nt][r], decay, dx * bv), sum = fmaf(next, cv, y);
        const bool in = WHOLE || n + r < d_state;  // (0 * infinity)
        h[nt][r] = in ? next : h[nt][r];
        y = in ? sum : y;
      }
      if (nt % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (not all loads of a row at once)
    }
    if constexpr (!STATES) {
      y += __shfl_xor(y, 16, 64);
      y += __shfl_xor(y, 32, 64);
      if (there && g == 0) w.y[t * a.y_rstride + li] = from_f32<T>(fmaf(skip, xv, y));
    }
  }
}

// STATES: first pass of a split call, the state every tile adds to a zero state.  Otherwise y (and the final states).
// WHOLE: head_dim is a multiple of 64, d_state is NP and the heads of a group are even: only rows can be missing.
template <typename T, int NP, bool STATES, bool WHOLE>
__global__ __launch_bounds__((ScanShape<T, NP, STATES>::THREADS), (ScanShape<T, NP, STATES>::WAVES)) void selective_scan_chunk_kernel(const mb_selective_scan_args a, const Split sp) {
  typedef ScanShape<T, NP, STATES> S;
  constexpr int V = 16 / sizeof(T), R = S::R, Q = S::Q, L = S::L, HB = S::HB, TT = S::TT, NT = S::NT, PB = S::PB, THREADS = S::THREADS;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  typename S::Lds& m = *(typename S::Lds*)lds_raw;

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63, g = lane >> 4, li = lane & 15;
  const Work<T> work = work_of<T, NP, STATES, WHOLE>(a, sp, blockIdx.x, wave);
  if (work.none) return;
  const int head_dim = a.head_dim, d_state = WHOLE ? NP : a.d_state_dim;
  const unsigned tile = work.tile;
  const int p0 = work.p0, head0 = work.head0, live = work.live, t0 = work.t0, t1 = work.t1, head = work.head, pw = work.columns, parts = work.parts;
  const T *xg = work.x, *bg = work.b, *cg = work.c;
  const long long dtg = work.dt;
  T* const yg = work.y;
  float* const pool = work.pool;
  const int hh = wave % HB, quarter = wave / HB;
  const bool mine = hh < live;
  f32x4 h[NT];
  start_of<T, NP, WHOLE>(work, head_dim, d_state, mine, lane, h);

  Stage<T, V, L, NP, THREADS> sb, sc;
  Stage<T, V, L, HB * PB, THREADS> sx;
  auto request = [&](int t, unsigned tid) {  // behind the last row: zeros without a load, so that no register has to keep an older chunk's values
    const int n = t1 - t;
    if constexpr (WHOLE) {
      sb.request(bg + t * a.b_rstride, (int)a.b_rstride, min(n, L), sb.offset(tid, (int)a.b_rstride), NP);
      if (!STATES) sc.request(cg + t * a.c_rstride, (int)a.c_rstride, min(n, L), sc.offset(tid, (int)a.c_rstride), NP);
      // two heads' columns p0 .. p0 + 63 are next to each other where head_dim is 64; else the second head's are head_dim - 64 further on
      const unsigned apart = (tid % sx.PER_ROW * V / PB) * (head_dim - PB) * (int)sizeof(T);
      sx.request(xg + t * a.x_rstride, (int)a.x_rstride, min(n, L), sx.offset(tid, (int)a.x_rstride) + apart, head_dim + PB);
    } else {
      auto col_n = [&](int c, int& left) {
        left = d_state - c;
        return c;
      };
      sb.request(bg + t * a.b_rstride, a.b_rstride, n, col_n);
      if (!STATES) sc.request(cg + t * a.c_rstride, a.c_rstride, n, col_n);
      sx.request(xg + t * a.x_rstride, a.x_rstride, n, [&](int c, int& left) {
        const int i = c / PB, p = c % PB;
        left = i < live ? head_dim - p0 - p : 0;
        return i * head_dim + p;
      });
    }
  };
  auto lay = [&](unsigned tid) {
    sb.template lay<R>(tid, [&](int q, unsigned r, unsigned c, const Vec<unsigned short, V>& v) { store_lds<V>(&m.b[q][r][c], v); });
    if constexpr (!STATES) sc.template lay<R>(tid, [&](int q, unsigned r, unsigned c, const Vec<unsigned short, V>& v) { store_lds<V>(&m.c[q][r][c], v); });
    sx.template lay<R>(tid, [&](int q, unsigned r, unsigned c, const Vec<unsigned short, V>& v) { store_lds<V>(&m.x[c / PB][q][r][S::x_col(r, c % PB)], v); });
  };
  // scalars of the heads, read once: inside the loop they would be loads behind its stores
  auto scalar = [&](const float* p, int at) { return __uint_as_float(__builtin_amdgcn_readfirstlane(p ? __float_as_uint(p[at]) : 0u)); };
  float A = scalar(a.d_a, head);
  const float bias = scalar(a.d_dt_bias, head);
  float skips[HB];
#pragma unroll
  for (int e = 0; e < HB; ++e) skips[e] = STATES ? 0.f : scalar(a.d_d, head0 + min(e, live - 1));
  double walked = 0.0;  // sum of d A over the tile so far: its decay
  // Everything of a chunk that depends on the step sizes alone, one lane per row.  Sums are fp64: a difference of two far prefixes keeps
  // its bits.  Exponents are base 2 from here on.
  float draw = 0.f;
  bool odd = !STATES && !(fabsf(skips[hh]) < INFINITY);  // something that the products cannot do: see the end
  auto request_step = [&](int t) { draw = lane < min(t1 - t, L) ? step_raw(a, dtg + (t + lane) * a.dt_rstride + head) : 0.f; };
  auto scalars = [&](int t, int to) {
    const bool row = lane < min(t1 - t, L);
    const float d = row ? step_of(a, draw, bias) : 0.f;
    asm("" : "+s"(A));  // (its fp64 copy is not worth registers of the whole loop)
    double s = row ? (double)d * ((double)A * 1.4426950408889634) : 0.0;  // log2(e)
    if (STATES && __any(s < -150.0)) walked = -INFINITY;  // a row whose own decay is zero
    s += row_shifted<1>(s);
    s += row_shifted<2>(s);
    s += row_shifted<4>(s);
    s += row_shifted<8>(s);  // from the start of the tile of 16 rows
    double rest = 0.0, sum[TT];  // of tile j
#pragma unroll
    for (int j = 0; j < TT; ++j) {
      sum[j] = from_lane(s, 16 * j + 15);
      if (g == j) rest = sum[j] - s;  // to the end of the tile
    }
    // prefixes that fp32 holds, growth that no product of factors takes out of it (NaN fails)
    if (__any(!(s > -1e38 && s < 28.0 && rest < 28.0 && fabsf(d) < INFINITY))) m.odd[hh][quarter] = 1;
    typename S::Head& o = m.head[to][hh];
    if (lane < L) {
      const float hi = (float)s;
      o.u[lane] = exp2_of(hi);
      o.w[lane] = exp2_of((float)rest) * d;
      o.hi[lane] = hi;
      o.lo[lane] = (float)(s - (double)hi);
      o.d[lane] = d;
    }
    // decays across whole tiles: products of theirs
    float by[TT], front = 1.f, back = 1.f;
#pragma unroll
    for (int j = 0; j < TT; ++j) by[j] = exp2_of((float)sum[j]);
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < TT; ++j) {
        o.front[j] = front;             // from the start of the chunk to the start of tile j
        o.back[TT - 1 - j] = back;      // from the end of that tile to the end of the chunk
        front *= by[j], back *= by[TT - 1 - j];
        float f = 1.f;                  // from the end of tile j to the start of tile k
#pragma unroll
        for (int k = j + 1; k < TT; ++k) {
          o.f[j][k] = f;
          f *= by[k];
        }
      }
      o.total = front;
    }
    if (STATES)
#pragma unroll
      for (int j = 0; j < TT; ++j) walked += sum[j];
  };

  if (WHOLE) request(t0, threadIdx.x);
  constexpr int HEADS = S::HEADS, FOUR = S::WPH;
  const bool stepper = mine && quarter == FOUR - 1;  // the wave of each head that does this, a chunk ahead of the others' products
  if (STATES ? mine : stepper) {
    m.odd[hh][quarter] = 0;
    const int first = STATES ? quarter : 0, next = STATES ? FOUR : 1;
    request_step(t0 + first * L);
    scalars(t0 + first * L, first);
    request_step(t0 + (first + next) * L);
  }
  int chunk = 0;
  for (int t = t0; t < t1; t += L, ++chunk) {
    const int now = chunk % HEADS;
    // The lane number is made new in every chunk: LDS addresses derived from it would otherwise be kept through the whole loop, in registers
    // that are not there.
    int fresh = lane;
    asm volatile("" : "+v"(fresh));
    const int g = fresh >> 4, li = fresh & 15, lane = fresh;
    const unsigned tid = (unsigned)(wave * 64 + fresh);
    if (!WHOLE) request(t, tid);  // masks and addresses of partial columns leave no registers to hold values through the products
    lay(tid);
    meet();
    const typename S::Head& hd = m.head[now][hh];
    if constexpr (STATES) {
      if (mine && chunk % FOUR == 0) {
        scalars(t + (FOUR + quarter) * L, (chunk + FOUR + quarter) % HEADS);
        request_step(t + (2 * FOUR + quarter) * L);
      }
    } else if (stepper) {
      scalars(t + L, now ^ 1);
      request_step(t + 2 * L);
    }

    f32x4 acc[TT];
    if constexpr (!STATES) {
      // G^T tiles (s tile i <= t tile j) dealt to the waves, and from each the M^T tiles of both heads: a diagonal tile to each of the first
      // TT waves, the others to the first 6 (the last two have the step sizes)
      constexpr int OFF = TT * (TT - 1) / 2;
      for (int k = wave < TT ? -1 : wave; k < OFF; k = k < 0 && wave < OFF ? wave : OFF) {
        const int j = k < 0 ? wave : k < 1 ? 1 : k < 3 ? 2 : 3, i = k < 0 ? wave : k - j * (j - 1) / 2;
        f32x4 gt = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NP; n += 32) {
          bf16x8 fa[R], fb[R];
#pragma unroll
          for (int q = 0; q < R; ++q) {
            fa[q] = *(const bf16x8*)&m.b[q][16 * i + li][n + 8 * g];
            fb[q] = *(const bf16x8*)&m.c[q][16 * j + li][n + 8 * g];
          }
          gt = mma<R, R, R>(fa, fb, gt);
          if (n % 64) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int e = 0; e < HB; ++e) {
          if (!WHOLE && e >= live) break;
          const typename S::Head& o = m.head[now][e];
          float v[4];
          if (i < j) {
            const f32x4 w = *(const f32x4*)&o.w[16 * i + 4 * g];
            const float u = o.u[16 * j + li] * o.f[i][j];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = gt[r] * (u * w[r]);
          } else {
            const f32x4 shi = *(const f32x4*)&o.hi[16 * i + 4 * g], slo = *(const f32x4*)&o.lo[16 * i + 4 * g];
            const f32x4 d = *(const f32x4*)&o.d[16 * i + 4 * g];
            const float thi = o.hi[16 * j + li], tlo = o.lo[16 * j + li], skip = skips[e];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              // the two differences of hi + lo parts are exact or as good as the exponent's own rounding
              float c = gt[r] * (exp2_of((thi - shi[r]) + (tlo - slo[r])) * d[r]), diagonal = fmaf(gt[r], d[r], skip);
              asm("" : "+v"(c), "+v"(diagonal));  // both are computed: selects, not branches per lane
              v[r] = 4 * g + r < li ? c : 4 * g + r == li ? diagonal : 0.f;
            }
          }
          float x0 = v[0], x1 = v[1], x2 = v[2], x3 = v[3];
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
            const u32x2 w = {pack_bf16(x0, x1), pack_bf16(x2, x3)};
            m.m[e][S::m_at(i, j, q, lane)] = __builtin_bit_cast(bf16x4, w);
            x0 -= __uint_as_float(w[0] << 16), x1 -= __uint_as_float(w[0] & 0xffff0000u);
            x2 -= __uint_as_float(w[1] << 16), x3 -= __uint_as_float(w[1] & 0xffff0000u);
          }
        }
      }
      // C h, scaled to each row's distance from the state
      if (mine) {
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        // the next operand is split between this one's products, a few vector instructions behind each
        bf16x8 fh[2][Q];
        auto split_h = [&](int n, bf16x8 (&to)[Q]) {
          const float v[8] = {h[n][0], h[n][1], h[n][2], h[n][3], h[n + 1][0], h[n + 1][1], h[n + 1][2], h[n + 1][3]};
          split<Q>(v, to);
        };
        split_h(0, fh[0]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          if (n + 2 < NT) split_h(n + 2, fh[n / 2 + 1 & 1]);
#pragma unroll
          for (int j = 0; j < TT; ++j) {
            bf16x8 fc[R];
#pragma unroll
            for (int q = 0; q < R; ++q) fc[q] = *(const bf16x8*)&m.c[q][16 * j + li][16 * n + 8 * g];
            acc[j] = mma<Q, R, Q>(fh[n / 2 & 1], fc, acc[j]);
          }
          behind_each<TT * S::CH_PAIRS, 3, TT * R, R>();
        }
#pragma unroll
        for (int j = 0; j < TT; ++j) {
          acc[j] *= hd.u[16 * j + li] * hd.front[j];
        }
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < TT; ++j) sum += acc[j][0];  // (a C that is not finite spoils its row in every column)
        odd |= !(fabsf(sum) < INFINITY);
      }
      meet();
    }
    if (mine) {
      auto read_x = [&](int k, bf16x8 (&to)[R]) {  // rows 32 k .. + 31 of this lane's column
#pragma unroll
        for (int q = 0; q < R; ++q) {
          const int r = 32 * k + 4 * g + (li >> 2), c = pw + 4 * (li & 3);
          to[q] = read_transposed(&m.x[hh][q][r][S::x_col(r, c)], &m.x[hh][q][r + 16][S::x_col(r + 16, c)]);
        }
      };
      auto scale_x = [&](int k, bf16x8 (&to)[3]) {  // c x
        const f32x4 c0 = *(const f32x4*)&hd.w[32 * k + 4 * g] * hd.back[2 * k], c1 = *(const f32x4*)&hd.w[32 * k + 16 + 4 * g] * hd.back[2 * k + 1];
        bf16x8 x[R];
        read_x(k, x);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float xv = value_of(x[R - 1], i);
#pragma unroll
          for (int q = R - 2; q >= 0; --q) xv += value_of(x[q], i);
          v[i] = (i < 4 ? c0[i & 3] : c1[i & 3]) * xv;
        }
        split<3>(v, to);
      };
      // h <- total h + B^T (c x)
      bf16x8 fs[2][3];
      scale_x(0, fs[0]);
      const float total = hd.total;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < L / 32; ++k) {
        if (k + 1 < L / 32) scale_x(k + 1, fs[k + 1 & 1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          bf16x8 fb[R];
#pragma unroll
          for (int q = 0; q < R; ++q) {
            const int r = 32 * k + 4 * g + (li >> 2), c = nt / 2 * 32 + nt % 2 * 4 + 8 * (li & 3);
            fb[q] = read_transposed(&m.b[q][r][c], &m.b[q][r + 16][c]);
          }
          if (k == 0) h[nt] *= total;
          h[nt] = mma<R, 3, 3>(fb, fs[k & 1], h[nt]);
        }
        if (k + 1 < L / 32) behind_each<NT * S::ST_PAIRS, 3, NT * 2 * R + 2 * R + 3, 4 * R>();
        else behind_each<NT * S::ST_PAIRS, 3, NT * 2 * R, 4 * R>();
      }
      // The next chunk is requested here, not before the products above: registers for both do not fit together, and the other workgroup
      // of the CU has work while it comes.
      __builtin_amdgcn_sched_barrier(0);
      if (WHOLE) request(t + L, tid);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (!STATES) {
        bf16x8 fx[L / 32][R];
#pragma unroll
        for (int k = 0; k < L / 32; ++k) read_x(k, fx[k]);
        const unsigned off_y = (li * (int)a.y_rstride + 4 * g) * (int)sizeof(T);
        // rows from the tile's end on are dropped by the descriptor's range check
        const __amdgpu_buffer_rsrc_t dy = tm_rsrc(yg + t * a.y_rstride, ((min(t1 - t, L) - 1) * (int)a.y_rstride + 16) * (int)sizeof(T));
#pragma unroll
        for (int j = 0; j < TT; ++j) {
#pragma unroll
          for (int k = 0; 2 * k < j; ++k) {
            bf16x8 fm[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) fm[q] = *(const bf16x8*)&m.m[hh][S::m_at(2 * k, j, q, lane)];
            acc[j] = mma<R, Q, Q>(fx[k], fm, acc[j]);
          }
          if (j % 2 == 0) {
            // 16 rows and 16 zeros, not the 16-row instruction: behind one of 32 rows on the same accumulators, with nothing between, it gave
            // wrong sums now and then
            bf16x8 fm[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) {
              const bf16x4 lo = m.m[hh][S::m_at(j, j, q, lane)];
              fm[q] = bf16x8{lo[0], lo[1], lo[2], lo[3], (__bf16)0.f, (__bf16)0.f, (__bf16)0.f, (__bf16)0.f};
            }
            acc[j] = mma<R, Q, Q>(fx[j / 2], fm, acc[j]);
          }
          if (j % 2) __builtin_amdgcn_sched_barrier(0);
        }
        // y^T tiles: row p = 4 g + i, column t = li
#pragma unroll
        for (int j = 0; j < TT; ++j) {
          Vec<T, 4> o;
#pragma unroll
          for (int r = 0; r < 4; ++r) o.v[r] = from_f32<T>(acc[j][r]);
          if constexpr (WHOLE) {
            typedef unsigned word __attribute__((ext_vector_type(sizeof(T))));
            const int more = 16 * j * (int)a.y_rstride * (int)sizeof(T);
            if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(word, o), dy, off_y, more, 0);
            else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(word, o), dy, off_y, more, 0);
          } else {
            const int row = t + 16 * j + li;
            if (row < t1) store_some<T, 4>(yg + row * a.y_rstride + 4 * g, o, head_dim - p0 - pw - 4 * g);
          }
        }
      }
    }
    meet();
  }

  if constexpr (STATES) {
    if (mine && lane == 0) m.walked[hh][quarter] = walked;  // each wave has summed up its own chunks
    meet();
  }
  if (!mine) return;
  if constexpr (STATES) {
    if (stepper && lane == 0) {
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < FOUR; ++i) sum += m.walked[hh][i];
      sp.decay[(long long)tile * a.heads + head] = sum == -INFINITY ? -0.f : exp2_of((float)sum);
    }
  }
  // Does this wave's result stand?  Products give NaN where the recurrence has an infinity, or a number: infinity - infinity between planes,
  // 0 * NaN in the half of M that is zero, 0 * infinity between the factors of a decay.  What of that comes from x, B, dt or the state in
  // front is in h for good, a C that is not finite was seen in C h, step sizes that the factors cannot do by the wave that made them.
  float spoilt = 0.f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 4; ++r) spoilt = fmaf(h[nt][r], 0.f, spoilt);
#pragma unroll
  for (int i = STATES ? 0 : FOUR - 1; i < FOUR; ++i) odd |= m.odd[hh][i] != 0;
  if (__any(odd || spoilt != 0.f)) walk_rows<T, NP, STATES, WHOLE>(h);
  if (!STATES && (!pool || work.part != parts - 1)) return;
  float* const to = STATES ? sp.state + ((long long)tile * a.heads + head) * ((long long)head_dim * d_state) : pool;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int p = p0 + pw + li, n = nt / 2 * 32 + 8 * g + nt % 2 * 4;
      if (WHOLE || p < head_dim)
        store_some<float, 4>(to + (long long)p * d_state + n, __builtin_bit_cast(Vec<float, 4>, h[nt]), WHOLE ? 4 : d_state - n);
    }
}

template <typename T, int NP, bool STATES, bool WHOLE> int launch_chunk(const mb_selective_scan_args& a, const Split& sp, hipStream_t s) {
  typedef ScanShape<T, NP, STATES> S;
  static_assert(sizeof(typename S::Lds) <= 160 * 1024, "a chunk has to fit LDS");
  const Rows rows = {a.d_cu_seqlens, a.d_valid, a.batch, a.t};
  const int per_group = a.heads / a.groups;
  const long long units = (long long)a.groups * cdiv(per_group, S::HB) * cdiv(a.head_dim, S::PB);
  const long long grid = (STATES ? sp.fronts : tiles_of(rows, sp.seg ? sp.seg : (a.t > 1 ? a.t : 1))) * units;
  MB_REQUIRE(launchable(grid, S::THREADS), "selective_scan: %d items of %d heads are too many for one launch", a.batch, a.heads);
  static std::atomic<unsigned long long> attr_done{0};  // per device: the attribute belongs to the function on the current device
  int dev = 0;
  MB_HIP(hipGetDevice(&dev));
  const unsigned long long bit = dev >= 0 && dev < 64 ? 1ull << dev : 0ull;
  if (!bit || !(attr_done.load(std::memory_order_acquire) & bit)) {
    MB_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&selective_scan_chunk_kernel<T, NP, STATES, WHOLE>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    attr_done.fetch_or(bit, std::memory_order_release);
  }
  hipLaunchKernelGGL((selective_scan_chunk_kernel<T, NP, STATES, WHOLE>), dim3((unsigned)grid), dim3(S::THREADS), sizeof(typename S::Lds), s, a, sp);
  MB_HIP(hipGetLastError());
  return MB_OK;
}

template <typename T, int NP> int chunk_by_shape(const mb_selective_scan_args& a, const Split& sp, bool states, hipStream_t s) {
  typedef ScanShape<T, NP, false> S;
  // WHOLE: no partial columns, rows apart from each other and words aligned (buffer accesses), a chunk within a descriptor's 31 bits
  auto fits = [&](const void* p, long long rstride, long long bstride, long long width) {
    return aligned(p, 4) && (rstride * (long long)sizeof(T)) % 4 == 0 && (a.d_cu_seqlens || bstride * (long long)sizeof(T) % 4 == 0) && rstride >= width &&
           rstride * S::L * (long long)sizeof(T) < (1ll << 31);
  };
  const long long wide = (long long)a.heads * a.head_dim, narrow = (long long)a.groups * a.d_state_dim;
  const bool whole = a.head_dim % S::PB == 0 && a.d_state_dim == NP && a.heads / a.groups % S::HB == 0 && fits(a.d_x, a.x_rstride, a.x_bstride, wide) &&
                     fits(a.d_y, a.y_rstride, a.y_bstride, wide) && fits(a.d_b, a.b_rstride, a.b_bstride, narrow) &&
                     fits(a.d_c, a.c_rstride, a.c_bstride, narrow);
  if (states) return whole ? launch_chunk<T, NP, true, true>(a, sp, s) : launch_chunk<T, NP, true, false>(a, sp, s);
  return whole ? launch_chunk<T, NP, false, true>(a, sp, s) : launch_chunk<T, NP, false, false>(a, sp, s);
}
template <typename T> int chunk_launch(const mb_selective_scan_args& a, const Split& sp, bool states, hipStream_t s) {
  if (a.d_state_dim <= 64) return chunk_by_shape<T, 64>(a, sp, states, s);
  if (a.d_state_dim <= 128) return chunk_by_shape<T, 128>(a, sp, states, s);
  return chunk_by_shape<T, 256>(a, sp, states, s);
}

// the kernels of one type each, in ssm_scan_{f32,f16,bf16}.hip
int scan_chunks_f32(const mb_selective_scan_args& a, const Split& sp, bool states, hipStream_t s);
int scan_chunks_f16(const mb_selective_scan_args& a, const Split& sp, bool states, hipStream_t s);
int scan_chunks_bf16(const mb_selective_scan_args& a, const Split& sp, bool states, hipStream_t s);

}  // namespace ssm
}  // namespace mb
