// The join of a block's branch with the residual stream, for gfx950, with
// the norms around it:
//
//   u = o rstd(o) post        (u = o without the post-norm)
//   r = stream_scale x + branch_scale gate u
//   y = r rstd(r) pre          rstd(v) = 1 / sqrt(mean v^2 + eps)
//
// and its gradient, for upstream dr and dy (h = v rstd(v)):
//
//   t = dr + rstd(r) (pre dy - h_r mean(pre dy h_r))
//   dx = stream_scale t                 dpre = sum over rows of dy h_r
//   e = branch_scale t                  dgate = sum over a gate row's rows of e u
//   do = rstd(o) (post gate e - h_o mean(post gate e h_o))   (gate e without)
//   dpost = sum over rows of gate e h_o
//
// Bound by HBM: the forward reads x and o and writes r and y, the gradient
// reads o, r, dr and dy and writes dx and do.  A row stays in registers
// between its load and its store, in 16-byte chunks at any address (8 bf16 or
// 4 fp32), on one to sixteen waves with 8 or 16 elements a thread; rows longer
// than that holds, and those shorter than a chunk, take the kernels at the end,
// which read them again from the caches.  (16 fp32 elements on sixteen waves, rows of
// 8193 to 16384, leave no registers for the next row's loads: 35 are spilled, 22 x
// 9152 9.8 us where 2 x 6144 takes 4.8.)  Sums are fp32; r is rounded once for
// its store and y comes from the unrounded r, so each output is rounded once.
// The gradient's sums over rows go to one partial row per block and a second
// launch adds those in order: no atomics, the same bits every time.
//
// 8192 x 4096 bf16 with other data in the caches: forward 55 us (268 MB, 4.9
// TB/s; a copy of as many bytes 54), gradient 92 us (403 MB, 4.4 TB/s).  The
// gradient is short of loads in flight: 16 elements on four waves take 222
// registers, two waves a SIMD, with the next row's loads ahead (8 elements on
// eight waves, one block a CU: 97; held to 128 registers for two, with spills:
// 177).
#pragma once

#include "common.h"
#include "../kargs.h"

using namespace bwpp;

namespace resnorm {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <class T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kPer = 4;  // per 16 bytes
  typedef uint32_t V __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ float get(const u32x4_t &v, int e) { return __uint_as_float(v[e]); }
  // Elements moved down by n, zeros behind them (n >= 4: all gone).
  static __device__ __forceinline__ u32x4_t down(u32x4_t v, uint32_t n) {
    const u32x4_t a = n & 1 ? u32x4_t{v[1], v[2], v[3], 0u} : v;
    const u32x4_t b = n & 2 ? u32x4_t{a[2], a[3], 0u, 0u} : a;
    return n < 4 ? b : u32x4_t{0u, 0u, 0u, 0u};
  }
  static __device__ __forceinline__ float one(float x) { return x; }
  static __device__ __forceinline__ float of(float x) { return x; }
};
template <>
struct Elem<uint16_t> {
  static constexpr int kPer = 8;
  typedef uint32_t V __attribute__((ext_vector_type(4), aligned(2)));
  static __device__ __forceinline__ float get(const u32x4_t &v, int e) {
    return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
  }
  static __device__ __forceinline__ u32x4_t down(u32x4_t v, uint32_t n) {
    const u32x4_t a = n & 1 ? u32x4_t{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16} : v;
    return n < 8 ? Elem<float>::down(a, n >> 1) : u32x4_t{0u, 0u, 0u, 0u};
  }
  static __device__ __forceinline__ float one(uint16_t x) { return bf16_bits_to_f32(x); }
  static __device__ __forceinline__ uint16_t of(float x) { return f32_to_bf16_bits(x); }
};

// One thread's share of a row: NC chunks, TPR threads apart.
template <class T, int NE, int TPR>
struct Part {
  static constexpr int E = Elem<T>::kPer, NC = NE / E;
  u32x4_t v[NC];

  __device__ __forceinline__ static uint32_t col(int j, int t) { return (uint32_t)(j * TPR + t) * E; }
  // A chunk that passes the row's end is read as the row's last E elements (cols
  // >= E); fix() moves it down, zeros behind the end, before the first use.
  __device__ __forceinline__ void load(const T *p, uint32_t cols, int t) {
#pragma unroll
    for (int j = 0; j < NC; ++j)
      v[j] = *reinterpret_cast<const typename Elem<T>::V *>(p + min(col(j, t), cols - E));
  }
  __device__ __forceinline__ void fix(uint32_t cols, int t) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const uint32_t c = col(j, t), from = min(c, cols - E);
      v[j] = Elem<T>::down(v[j], c - from);
    }
  }
  __device__ __forceinline__ void load_fixed(const T *p, uint32_t cols, int t) {
    load(p, cols, t);
    fix(cols, t);
  }
  __device__ __forceinline__ void fill_one() {
#pragma unroll
    for (int j = 0; j < NC; ++j)
      v[j] = E == 4 ? u32x4_t{0x3f800000u, 0x3f800000u, 0x3f800000u, 0x3f800000u}
                    : u32x4_t{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < NC; ++j) v[j] = u32x4_t{0u, 0u, 0u, 0u};
  }
  // Keeps the packed values: unpacked ahead of a loop they would fill twice
  // the registers.
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t x = v[j][e];
        asm volatile("" : "+v"(x));
        v[j][e] = x;
      }
  }
  __device__ __forceinline__ float at(int i) const { return Elem<T>::get(v[i / E], i % E); }

  __device__ __forceinline__ static void store(T *p, const float (&x)[NE], uint32_t cols, int t) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const uint32_t c = col(j, t);
      if (c + E <= cols) {
        u32x4_t o;
        if constexpr (E == 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = __float_as_uint(x[j * E + e]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = pack_bf16x2(x[j * E + 2 * e], x[j * E + 2 * e + 1]);
        }
        *reinterpret_cast<typename Elem<T>::V *>(p + c) = o;
      } else if (c < cols) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < cols) p[c + e] = Elem<T>::of(x[j * E + e]);
      }
    }
  }
  // fp32 row (partials; 4-byte aligned).
  __device__ __forceinline__ static void store_f32(float *p, const float (&x)[NE], uint32_t cols, int t) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const uint32_t c = col(j, t);
      if (c + E <= cols) {
#pragma unroll
        for (int e = 0; e < E; e += 4)
          store4(p + c + e, make_float4(x[j * E + e], x[j * E + e + 1], x[j * E + e + 2], x[j * E + e + 3]));
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < cols) p[c + e] = x[j * E + e];
      }
    }
  }
};

// Sums over the waves of a row.  Every call of a block uses the next of four
// slots: a wave can be one barrier ahead of another, never two.
template <int WPR, int N>
struct RowSum {
  float (*slots)[N][16];
  uint32_t next = 0;
  __device__ __forceinline__ void operator()(float (&s)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = wave_sum(s[i]);
    if constexpr (WPR > 1) {
      float (*sl)[16] = slots[next];
      next = (next + 1) & 3u;
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) sl[i][threadIdx.x >> 6] = s[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float p[WPR];
#pragma unroll
        for (int w = 0; w < WPR; ++w) p[w] = sl[i][w];
#pragma unroll
        for (int d = 1; d < WPR; d *= 2)
#pragma unroll
          for (int w = 0; w + d < WPR; w += 2 * d) p[w] += p[w + d];
        s[i] = p[0];
      }
    }
  }
};

__device__ __forceinline__ float rstd(float sum, const BwppResNormArgs &a) {
  return 1.0f / sqrtf(sum / (float)a.cols + a.eps);
}

// branch_scale gate post of this thread's columns, in fp32.
template <class T, int NE, int TPR>
__device__ __forceinline__ void gate_post(float (&pg)[NE], const BwppResNormArgs &a, const Part<T, NE, TPR> &g, int t) {
  Part<T, NE, TPR> post;
  if (a.post_norm && a.post) post.load_fixed(static_cast<const T *>(a.post), a.cols, t);
  else post.fill_one();
#pragma unroll
  for (int i = 0; i < NE; ++i) pg[i] = a.branch_scale * g.at(i) * post.at(i);
}

template <class T, int NE, int WPR>
__device__ __forceinline__ void forward(const BwppResNormArgs &a) {
  constexpr int TPR = 64 * WPR, RPB = WPR == 1 ? 4 : 1;
  using P = Part<T, NE, TPR>;
  __shared__ float slots[4][1][16];
  RowSum<WPR, 1> sum{slots};
  const int t = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const T *x = static_cast<const T *>(a.x), *o = static_cast<const T *>(a.o), *gate = static_cast<const T *>(a.gate);
  P pre, g, px, po;
  pre.fill_one();
  g.fill_one();
  if (a.y && a.pre) pre.load_fixed(static_cast<const T *>(a.pre), a.cols, t);
  const bool gated = gate && a.gate_rows;  // a gate row of its own for some rows
  const bool edge = a.cols < (uint32_t)(NE * TPR);
  if (gate && !gated) g.load_fixed(gate, a.cols, t);
  float pg[NE];
  if (!gated) gate_post(pg, a, g, t);
  const uint64_t step = (uint64_t)gridDim.x * RPB;
  uint64_t row = (uint64_t)blockIdx.x * RPB + (WPR == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
  if (row < a.rows) {
    px.load(x + row * a.ldx, a.cols, t);
    po.load(o + row * a.ldo, a.cols, t);
    if (gated) g.load(gate + row / a.gate_rows * a.ldg, a.cols, t);
  }
  for (; row < a.rows; row += step) {
    // The next row is on its way while this one is reduced (in place too: a
    // row is read by the threads that write it, and by no others).
    P nx, no, ng = g;
    const uint64_t nr = row + step < a.rows ? row + step : row;
    nx.load(x + nr * a.ldx, a.cols, t);
    no.load(o + nr * a.ldo, a.cols, t);
    if (gated) {
      ng.load(gate + nr / a.gate_rows * a.ldg, a.cols, t);
      if (edge) g.fix(a.cols, t);
      gate_post(pg, a, g, t);
    }
    if (edge) {
      px.fix(a.cols, t);
      po.fix(a.cols, t);
    }
    float s[1] = {0.0f}, r[NE], io = 1.0f;
    if (a.post_norm) {
#pragma unroll
      for (int i = 0; i < NE; ++i) s[0] = fmaf(po.at(i), po.at(i), s[0]);
      sum(s);
      io = rstd(s[0], a);
    }
    s[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      r[i] = fmaf(pg[i] * po.at(i), io, a.stream_scale * px.at(i));
      s[0] = fmaf(r[i], r[i], s[0]);
    }
    P::store(static_cast<T *>(a.ro) + row * a.ldx, r, a.cols, t);
    if (a.y) {
      sum(s);
      const float ir = rstd(s[0], a);
#pragma unroll
      for (int i = 0; i < NE; ++i) r[i] = r[i] * ir * pre.at(i);
      P::store(static_cast<T *>(a.y) + row * a.ldy, r, a.cols, t);
    }
    px = nx;
    po = no;
    g = ng;
  }
}

// One worker's rows r0, r0 + step, .. below r1: see BwppResNormArgs.  Blocks that
// share a group take its rows in turn, so that all of them stream through one
// part of memory (a run of rows each: 5 % slower at 8192 x 4096).
__device__ __forceinline__ void worker_rows(const BwppResNormArgs &a, uint64_t w, uint64_t &r0, uint64_t &r1,
                                            uint64_t &step) {
  step = 1;
  if (w >= a.workers) {
    r0 = r1 = a.rows;
  } else if (a.split > 1) {
    const uint64_t g = w / a.split;
    step = a.split;
    r1 = min((g + 1) * a.group, (uint64_t)a.rows);
    r0 = min(g * a.group + w % a.split, r1);
  } else {
    r0 = min(w * a.span, (uint64_t)a.rows);
    r1 = min(r0 + a.span, (uint64_t)a.rows);
  }
}

// One partial row per block: of one wave's rows each (WPR = 1) the four sums are
// added in LDS first.
template <class P, int NE, int WPR>
__device__ __forceinline__ void store_part(float *part, float (&x)[NE], uint32_t cols, int t, float *lds) {
  if (!part) return;
  part += (uint64_t)blockIdx.x * cols;
  if constexpr (WPR == 1) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NE; ++i) lds[(wave * NE + i) * 64 + t] = x[i];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      x[i] = (lds[i * 64 + t] + lds[(NE + i) * 64 + t]) + (lds[(2 * NE + i) * 64 + t] + lds[(3 * NE + i) * 64 + t]);
  }
  P::store_f32(part, x, cols, t);
}

// With pg = branch_scale gate post (a column's, while the gate row lasts):
//   t   = dr + rstd(r) pre dy - k r        k = rstd(r)^2 mean(pre dy h_r)
//   do  = rstd(o) pg t - l o               l = rstd(o)^2 mean(pg t h_o)
//   q   = sum over a gate row's rows of t h_o, from which dgate = branch_scale
//         post q and dpost adds branch_scale gate q: one sum of columns a row
// instead of two, and 23 instructions an element.
template <class T, int NE, int WPR>
__device__ __forceinline__ void gradient(const BwppResNormArgs &a) {
  constexpr int TPR = 64 * WPR, RPB = WPR == 1 ? 4 : 1;
  using P = Part<T, NE, TPR>;
  __shared__ float slots[4][3][16];
  __shared__ float slots1[4][1][16];
  RowSum<WPR, 3> sum3{slots};
  RowSum<WPR, 1> sum1{slots1};
  const int t = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  __shared__ float lds[WPR == 1 ? 4 * NE * 64 : 1];
  // A worker is a block, whose four waves take its rows in turn (WPR = 1, split
  // gate rows), or a wave or block with whole gate rows of its own.
  const uint32_t wave = WPR == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const bool turns = RPB > 1 && a.split > 1;
  uint64_t row, end, step;
  worker_rows(a, turns ? blockIdx.x : (uint64_t)blockIdx.x * RPB + wave, row, end, step);
  if (turns) {
    row += wave * step;
    step *= RPB;
  }
  const T *o = static_cast<const T *>(a.o), *r = static_cast<const T *>(a.r), *gate = static_cast<const T *>(a.gate);
  const T *dr = static_cast<const T *>(a.dr), *dy = static_cast<const T *>(a.dy);
  float apre[NE], apost[NE], q[NE], pg[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) apre[i] = apost[i] = q[i] = 0.0f;
  P pre, po, pr, pd, py;
  pre.fill_one();
  if (a.pre) pre.load_fixed(static_cast<const T *>(a.pre), a.cols, t);
  const uint64_t gr = a.gate_rows ? a.gate_rows : a.rows;  // rows of a gate row
  uint64_t gate_row = 0, gate_end = 0;                     // the present one and its end
  auto load_gate = [&](P &g) {
    if (gate) g.load_fixed(gate + gate_row * a.ldg, a.cols, t);
    else g.fill_one();
  };
  auto load = [&](P &lo, P &lr, P &ld, P &ly, uint64_t i) {
    lo.load(o + i * a.ldo, a.cols, t);
    lr.load(r + i * a.ldx, a.cols, t);
    if (dr) ld.load(dr + i * a.ldx, a.cols, t);
    else ld.zero();
    if (dy) ly.load(dy + i * a.ldy, a.cols, t);
    else ly.zero();
  };
  if (row < end) load(po, pr, pd, py, row);
  for (; row < end; row += step) {
    if (row >= gate_end) {
      gate_row = row / gr;
      gate_end = (gate_row + 1) * gr;
      P g;
      load_gate(g);
      gate_post(pg, a, g, t);
    }
    // bf16: the next row is on its way while this one is reduced.
    constexpr bool kAhead = sizeof(T) == 2;
    P no, nr, nd, ny;
    if constexpr (kAhead) load(no, nr, nd, ny, row + step < end ? row + step : row);
    if (a.cols < (uint32_t)(NE * TPR)) {
      po.fix(a.cols, t);
      pr.fix(a.cols, t);
      if (dr) pd.fix(a.cols, t);
      if (dy) py.fix(a.cols, t);
    }
    if constexpr (sizeof(T) == 2) pre.pin();
    float s3[3] = {0.0f, 0.0f, 0.0f};  // r^2, o^2, pre dy r
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      s3[0] = fmaf(pr.at(i), pr.at(i), s3[0]);
      s3[1] = fmaf(po.at(i), po.at(i), s3[1]);
      s3[2] = fmaf(pre.at(i) * py.at(i), pr.at(i), s3[2]);
    }
    sum3(s3);
    const float ir = dy ? rstd(s3[0], a) : 0.0f, io = a.post_norm ? rstd(s3[1], a) : 1.0f;
    const float k = s3[2] * ir * ir * ir / (float)a.cols;
    float d[NE], out[NE], s1[1] = {0.0f};  // d: t of the row
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      d[i] = fmaf(-k, pr.at(i), fmaf(ir, pre.at(i) * py.at(i), pd.at(i)));
      apre[i] = fmaf(py.at(i), pr.at(i) * ir, apre[i]);
      const float to = d[i] * po.at(i);
      q[i] = fmaf(to, io, q[i]);
      s1[0] = fmaf(pg[i], to, s1[0]);
      out[i] = a.stream_scale * d[i];
    }
    if (a.dx) P::store(static_cast<T *>(a.dx) + row * a.ldx, out, a.cols, t);
    if (a.dout) {
      float l = 0.0f;
      if (a.post_norm) {
        sum1(s1);
        l = s1[0] * io * io * io / (float)a.cols;
      }
#pragma unroll
      for (int i = 0; i < NE; ++i) out[i] = fmaf(pg[i] * d[i], io, -l * po.at(i));
      P::store(static_cast<T *>(a.dout) + row * a.ldo, out, a.cols, t);
    }
    if (row + step >= gate_end || row + step >= end) {  // the gate row's last row here
      P g, post;
      load_gate(g);
      if (a.post_norm && a.post) post.load_fixed(static_cast<const T *>(a.post), a.cols, t);
      else post.fill_one();
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        const float bq = a.branch_scale * q[i];
        apost[i] = fmaf(g.at(i), bq, apost[i]);
        q[i] = post.at(i) * bq;
      }
      // Where dgate's rows are split over blocks, this is the only one of the
      // block's and its sum stays in q.
      if (!a.part_gate) {
        if (a.dgate) P::store(static_cast<T *>(a.dgate) + row / a.group * a.ldg, q, a.cols, t);
#pragma unroll
        for (int i = 0; i < NE; ++i) q[i] = 0.0f;
      }
    }
    if constexpr (kAhead) {
      po = no;
      pr = nr;
      pd = nd;
      py = ny;
    } else if (row + step < end) {
      load(po, pr, pd, py, row + step);
    }
  }
  store_part<P, NE, WPR>(a.part_pre, apre, a.cols, t, lds);
  store_part<P, NE, WPR>(a.part_post, apost, a.cols, t, lds);
  store_part<P, NE, WPR>(a.part_gate, q, a.cols, t, lds);
}

// Any row length: one block per row (forward) or worker (gradient), which
// reads its rows again for each step.
constexpr int kGenWaves = 8, kGenNT = 64 * kGenWaves;

template <class T>
__device__ __forceinline__ void forward_any(const BwppResNormArgs &a) {
  __shared__ float slots[4][1][16];
  RowSum<kGenWaves, 1> sum{slots};
  const T *post = static_cast<const T *>(a.post), *pre = static_cast<const T *>(a.pre);
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.ldx, *o = static_cast<const T *>(a.o) + row * a.ldo;
    const T *g = a.gate ? static_cast<const T *>(a.gate) + (a.gate_rows ? row / a.gate_rows * a.ldg : 0) : nullptr;
    T *ro = static_cast<T *>(a.ro) + row * a.ldx;
    float s[1] = {0.0f}, io = 1.0f;
    if (a.post_norm) {
      for (uint32_t c = threadIdx.x; c < a.cols; c += kGenNT) {
        const float v = Elem<T>::one(o[c]);
        s[0] = fmaf(v, v, s[0]);
      }
      sum(s);
      io = rstd(s[0], a);
    }
    auto join = [&](uint32_t c) {
      const float gv = g ? Elem<T>::one(g[c]) : 1.0f, pv = a.post_norm && post ? Elem<T>::one(post[c]) : 1.0f;
      return fmaf(a.branch_scale * gv, Elem<T>::one(o[c]) * io * pv, a.stream_scale * Elem<T>::one(x[c]));
    };
    s[0] = 0.0f;
    if (a.y) {
      for (uint32_t c = threadIdx.x; c < a.cols; c += kGenNT) {
        const float r = join(c);
        s[0] = fmaf(r, r, s[0]);
      }
      sum(s);
    }
    const float ir = a.y ? rstd(s[0], a) : 0.0f;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kGenNT) {
      const float r = join(c);
      ro[c] = Elem<T>::of(r);
      if (a.y) static_cast<T *>(a.y)[row * a.ldy + c] = Elem<T>::of(r * ir * (pre ? Elem<T>::one(pre[c]) : 1.0f));
    }
  }
}

template <class T>
__device__ __forceinline__ void gradient_any(const BwppResNormArgs &a) {
  __shared__ float slots[4][3][16];
  __shared__ float slots1[4][1][16];
  RowSum<kGenWaves, 3> sum3{slots};
  RowSum<kGenWaves, 1> sum1{slots1};
  const T *post = a.post_norm ? static_cast<const T *>(a.post) : nullptr, *pre = static_cast<const T *>(a.pre);
  const uint64_t w = blockIdx.x;
  uint64_t row, end, step;
  worker_rows(a, w, row, end, step);
  // Partial rows are summed in memory, each column by one thread.
  float *parts[3] = {a.part_pre, a.part_post, a.part_gate};
  for (float *p : parts)
    if (p)
      for (uint32_t c = threadIdx.x; c < a.cols; c += kGenNT) p[w * a.cols + c] = 0.0f;
  for (; row < end; row += step) {
    const T *o = static_cast<const T *>(a.o) + row * a.ldo, *r = static_cast<const T *>(a.r) + row * a.ldx;
    const T *g = a.gate ? static_cast<const T *>(a.gate) + (a.gate_rows ? row / a.gate_rows * a.ldg : 0) : nullptr;
    const T *dr = a.dr ? static_cast<const T *>(a.dr) + row * a.ldx : nullptr;
    const T *dy = a.dy ? static_cast<const T *>(a.dy) + row * a.ldy : nullptr;
    auto one = [](const T *p, uint32_t c, float none) { return p ? Elem<T>::one(p[c]) : none; };
    float s3[3] = {0.0f, 0.0f, 0.0f};
    for (uint32_t c = threadIdx.x; c < a.cols; c += kGenNT) {
      const float rv = one(r, c, 0.0f), ov = one(o, c, 0.0f);
      s3[0] = fmaf(rv, rv, s3[0]);
      s3[1] = fmaf(ov, ov, s3[1]);
      s3[2] = fmaf(one(pre, c, 1.0f) * one(dy, c, 0.0f), rv, s3[2]);
    }
    sum3(s3);
    const float ir = dy ? rstd(s3[0], a) : 0.0f, io = a.post_norm ? rstd(s3[1], a) : 1.0f;
    const float mr = s3[2] * ir / (float)a.cols;
    auto t_at = [&](uint32_t c) {
      const float hr = one(r, c, 0.0f) * ir;
      return fmaf(ir, fmaf(one(pre, c, 1.0f), one(dy, c, 0.0f), -hr * mr), one(dr, c, 0.0f));
    };
    float s1[1] = {0.0f};
    if (a.dout && a.post_norm) {
      for (uint32_t c = threadIdx.x; c < a.cols; c += kGenNT)
        s1[0] = fmaf(one(post, c, 1.0f) * (one(g, c, 1.0f) * (a.branch_scale * t_at(c))), one(o, c, 0.0f) * io, s1[0]);
      sum1(s1);
    }
    const float mo = s1[0] / (float)a.cols;
    const bool flush = a.split == 1 && (row + 1 == a.rows || (row + 1) % a.group == 0);
    for (uint32_t c = threadIdx.x; c < a.cols; c += kGenNT) {
      const float tt = t_at(c), e = a.branch_scale * tt, ge = one(g, c, 1.0f) * e, ho = one(o, c, 0.0f) * io;
      const float pv = one(post, c, 1.0f), dyv = one(dy, c, 0.0f), hr = one(r, c, 0.0f) * ir;
      if (a.dx) static_cast<T *>(a.dx)[row * a.ldx + c] = Elem<T>::of(a.stream_scale * tt);
      if (a.dout) static_cast<T *>(a.dout)[row * a.ldo + c] = Elem<T>::of(a.post_norm ? io * fmaf(pv, ge, -ho * mo) : ge);
      if (a.part_pre) a.part_pre[w * a.cols + c] = fmaf(dyv, hr, a.part_pre[w * a.cols + c]);
      if (a.part_post) a.part_post[w * a.cols + c] = fmaf(ge, ho, a.part_post[w * a.cols + c]);
      if (a.part_gate) {
        const float v = fmaf(e, ho * pv, a.part_gate[w * a.cols + c]);
        a.part_gate[w * a.cols + c] = flush ? 0.0f : v;
        if (flush) static_cast<T *>(a.dgate)[row / a.group * a.ldg + c] = Elem<T>::of(v);
      }
    }
  }
}

// Partial rows -> weight gradients: blocks of 64 columns; grid y 0: dpre, 1:
// dpost, 2 + g: dgate of gate row g (its `split` workers).  Sixteen waves take a
// run of the rows each, eight loads in flight, then their sums are added in order.
template <class T>
__device__ __forceinline__ void finish(const BwppResNormArgs &a) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t c = blockIdx.x * 64 + lane, which = blockIdx.y;
  const float *part = which == 0 ? a.part_pre : which == 1 ? a.part_post : a.part_gate;
  T *out = static_cast<T *>(which == 0 ? a.dpre : which == 1 ? a.dpost : a.dgate);
  if (!part || !out) return;
  uint32_t n = a.nparts;
  if (which >= 2) {
    part += (uint64_t)(which - 2) * a.split * a.cols;
    out += (uint64_t)(which - 2) * a.ldg;
    n = a.split;
  }
  const uint32_t run = (n + 15) / 16, p0 = min(wave * run, n), p1 = min(p0 + run, n);
  float v[8] = {};
  if (c < a.cols) {
    uint32_t p = p0;
    for (; p + 8 <= p1; p += 8)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += part[(uint64_t)(p + i) * a.cols + c];
    for (; p < p1; ++p) v[0] += part[(uint64_t)p * a.cols + c];
  }
  s[wave][lane] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  __syncthreads();
  if (wave != 0 || c >= a.cols) return;
  float sum = s[0][lane];
#pragma unroll
  for (int i = 1; i < 16; ++i) sum += s[i][lane];
  out[c] = Elem<T>::of(sum);
}

#define BWPP_RESNORM(TN, T, NE, WPR)                                                                           \
  extern "C" __global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void bwpp_resnorm_##TN##_n##NE##_w##WPR( \
      const BwppResNormArgs a) {                                                                               \
    forward<T, NE, WPR>(a);                                                                                    \
  }
#define BWPP_RESNORM_GRAD(TN, T, NE, WPR)                                                                           \
  extern "C" __global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void bwpp_resnorm_grad_##TN##_n##NE##_w##WPR( \
      const BwppResNormArgs a) {                                                                                    \
    gradient<T, NE, WPR>(a);                                                                                        \
  }
#define BWPP_RESNORM_ALL(TN, T)                                                                                \
  BWPP_RESNORM(TN, T, 8, 1)                                                                                    \
  BWPP_RESNORM(TN, T, 8, 2)                                                                                    \
  BWPP_RESNORM(TN, T, 8, 4)                                                                                    \
  BWPP_RESNORM(TN, T, 8, 8)                                                                                    \
  BWPP_RESNORM(TN, T, 8, 16)                                                                                   \
  BWPP_RESNORM(TN, T, 16, 16)                                                                                  \
  BWPP_RESNORM_GRAD(TN, T, 8, 1)                                                                            \
  BWPP_RESNORM_GRAD(TN, T, 16, 1)                                                                           \
  BWPP_RESNORM_GRAD(TN, T, 16, 2)                                                                           \
  BWPP_RESNORM_GRAD(TN, T, 16, 4)                                                                           \
  BWPP_RESNORM_GRAD(TN, T, 8, 8)                                                                            \
  BWPP_RESNORM_GRAD(TN, T, 16, 8)                                                                           \
  extern "C" __global__ __launch_bounds__(kGenNT) void bwpp_resnorm_##TN##_any(const BwppResNormArgs a) {      \
    forward_any<T>(a);                                                                                         \
  }                                                                                                            \
  extern "C" __global__ __launch_bounds__(kGenNT) void bwpp_resnorm_grad_##TN##_any(const BwppResNormArgs a) { \
    gradient_any<T>(a);                                                                                        \
  }                                                                                                            \
  extern "C" __global__ __launch_bounds__(1024) void bwpp_resnorm_finish_##TN(const BwppResNormArgs a) { finish<T>(a); }
BWPP_RESNORM_ALL(bf16, uint16_t)
BWPP_RESNORM_ALL(f32, float)

}  // namespace resnorm
