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
// 4 fp32), on one wave (up to 512 columns) to eight (4096 and more, up to four
// times 8 elements a thread); longer rows take the kernels at the end, which
// read them again from the caches.  Sums are fp32; r is rounded once for its
// store and y comes from the unrounded r, so each output is rounded once.
// The gradient's sums over rows go to one partial row per worker and a second
// launch adds those in order: no atomics, the same bits every time.
#include "common.h"
#include "../kargs.h"

using namespace bwpp;

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <class T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kPer = 4;  // per 16 bytes
  typedef uint32_t V __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ float get(const u32x4_t &v, int e) { return __uint_as_float(v[e]); }
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
  static __device__ __forceinline__ float one(uint16_t x) { return bf16_bits_to_f32(x); }
  static __device__ __forceinline__ uint16_t of(float x) { return f32_to_bf16_bits(x); }
};

// One thread's share of a row: NC chunks, TPR threads apart.
template <class T, int NE, int TPR>
struct Part {
  static constexpr int E = Elem<T>::kPer, NC = NE / E;
  u32x4_t v[NC];

  __device__ __forceinline__ static uint32_t col(int j, int t) { return (uint32_t)(j * TPR + t) * E; }
  __device__ __forceinline__ void load(const T *p, uint32_t cols, int t) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const uint32_t c = col(j, t);
      v[j] = u32x4_t{0u, 0u, 0u, 0u};
      if (c + E <= cols) {
        v[j] = *reinterpret_cast<const typename Elem<T>::V *>(p + c);
      } else if (c < cols) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < cols) {
            const uint32_t b = __float_as_uint(Elem<T>::one(p[c + e]));
            if constexpr (E == 4) v[j][e] = b;
            else v[j][e >> 1] |= e & 1 ? b : b >> 16;
          }
      }
    }
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

template <class T, int NE, int WPR>
__device__ __forceinline__ void forward(const BwppResNormArgs &a) {
  constexpr int TPR = 64 * WPR, RPB = WPR == 1 ? 4 : 1;
  using P = Part<T, NE, TPR>;
  __shared__ float slots[4][1][16];
  RowSum<WPR, 1> sum{slots};
  const int t = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const T *x = static_cast<const T *>(a.x), *o = static_cast<const T *>(a.o), *gate = static_cast<const T *>(a.gate);
  P post, pre, g, px, po;
  post.fill_one();
  pre.fill_one();
  g.fill_one();
  if (a.post_norm && a.post) post.load(static_cast<const T *>(a.post), a.cols, t);
  if (a.y && a.pre) pre.load(static_cast<const T *>(a.pre), a.cols, t);
  const bool gated = gate && a.gate_rows;  // a gate row of its own for some rows
  if (gate && !gated) g.load(gate, a.cols, t);
  const uint64_t step = (uint64_t)gridDim.x * RPB;
  uint64_t row = (uint64_t)blockIdx.x * RPB + (WPR == 1 ? threadIdx.x >> 6 : 0);
  if (row < a.rows) {
    px.load(x + row * a.ldx, a.cols, t);
    po.load(o + row * a.ldo, a.cols, t);
    if (gated) g.load(gate + row / a.gate_rows * a.ldg, a.cols, t);
  }
  for (; row < a.rows; row += step) {
    // The next row is on its way while this one is reduced (in place too: a
    // row is read by the threads that write it, and by no others).
    P nx, no, ng = g;
    const uint64_t nr = row + step;
    if (nr < a.rows) {
      nx.load(x + nr * a.ldx, a.cols, t);
      no.load(o + nr * a.ldo, a.cols, t);
      if (gated) ng.load(gate + nr / a.gate_rows * a.ldg, a.cols, t);
    }
    float s[1] = {0.0f}, r[NE], io = 1.0f;
    if (a.post_norm) {
#pragma unroll
      for (int i = 0; i < NE; ++i) s[0] = fmaf(po.at(i), po.at(i), s[0]);
      sum(s);
      io = rstd(s[0], a);
    }
    const float bs = a.branch_scale;
    s[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      r[i] = fmaf(bs * g.at(i), po.at(i) * io * post.at(i), a.stream_scale * px.at(i));
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

// One worker's rows [r0, r1): see BwppResNormArgs.
__device__ __forceinline__ bool worker_rows(const BwppResNormArgs &a, uint64_t w, uint64_t &r0, uint64_t &r1) {
  if (w >= a.workers) return false;
  if (a.split > 1) {
    const uint64_t g = w / a.split, k = w % a.split, end = min((g + 1) * a.group, (uint64_t)a.rows);
    r0 = min(g * a.group + k * a.span, end);
    r1 = min(r0 + a.span, end);
  } else {
    r0 = min(w * a.span, (uint64_t)a.rows);
    r1 = min(r0 + a.span, (uint64_t)a.rows);
  }
  return true;
}

template <class T, int NE, int WPR>
__device__ __forceinline__ void gradient(const BwppResNormArgs &a) {
  constexpr int TPR = 64 * WPR, RPB = WPR == 1 ? 4 : 1;
  using P = Part<T, NE, TPR>;
  __shared__ float slots[4][3][16];
  __shared__ float slots1[4][1][16];
  RowSum<WPR, 3> sum3{slots};
  RowSum<WPR, 1> sum1{slots1};
  const int t = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const uint64_t w = (uint64_t)blockIdx.x * RPB + (WPR == 1 ? threadIdx.x >> 6 : 0);
  uint64_t row, end;
  if (!worker_rows(a, w, row, end)) return;  // WPR > 1: the whole block
  const T *o = static_cast<const T *>(a.o), *r = static_cast<const T *>(a.r), *gate = static_cast<const T *>(a.gate);
  const T *dr = static_cast<const T *>(a.dr), *dy = static_cast<const T *>(a.dy);
  P post, pre, g;
  post.fill_one();
  pre.fill_one();
  g.fill_one();
  if (a.post_norm && a.post) post.load(static_cast<const T *>(a.post), a.cols, t);
  if (a.pre) pre.load(static_cast<const T *>(a.pre), a.cols, t);
  const bool gated = gate && a.gate_rows;
  if (gate && !gated) g.load(gate, a.cols, t);
  float apre[NE], apost[NE], agate[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) apre[i] = apost[i] = agate[i] = 0.0f;
  P po, pr, pd, py;
  auto load = [&](P &lo, P &lr, P &ld, P &ly, P &lg, uint64_t i) {
    lo.load(o + i * a.ldo, a.cols, t);
    lr.load(r + i * a.ldx, a.cols, t);
    if (dr) ld.load(dr + i * a.ldx, a.cols, t);
    else ld.zero();
    if (dy) ly.load(dy + i * a.ldy, a.cols, t);
    else ly.zero();
    if (gated) lg.load(gate + i / a.gate_rows * a.ldg, a.cols, t);
  };
  if (row < end) load(po, pr, pd, py, g, row);
  for (; row < end; ++row) {
    // (sixteen waves leave 128 registers a thread, too few for a second row)
    constexpr bool kAhead = WPR < 16;
    P no, nr, nd, ny, ng = g;
    if constexpr (kAhead)
      if (row + 1 < end) load(no, nr, nd, ny, ng, row + 1);
    float s3[3] = {0.0f, 0.0f, 0.0f};  // r^2, o^2, pre dy r
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      s3[0] = fmaf(pr.at(i), pr.at(i), s3[0]);
      s3[1] = fmaf(po.at(i), po.at(i), s3[1]);
      s3[2] = fmaf(pre.at(i) * py.at(i), pr.at(i), s3[2]);
    }
    sum3(s3);
    const float ir = dy ? rstd(s3[0], a) : 0.0f, io = a.post_norm ? rstd(s3[1], a) : 1.0f;
    const float mr = s3[2] * ir / (float)a.cols;  // mean(pre dy h_r)
    float d[NE], s1[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const float hr = pr.at(i) * ir, ho = po.at(i) * io;
      const float tt = fmaf(ir, fmaf(pre.at(i), py.at(i), -hr * mr), pd.at(i));
      d[i] = a.stream_scale * tt;
      apre[i] = fmaf(py.at(i), hr, apre[i]);
      const float e = a.branch_scale * tt, ge = g.at(i) * e;
      agate[i] = fmaf(e, ho * post.at(i), agate[i]);
      apost[i] = fmaf(ge, ho, apost[i]);
      s1[0] = fmaf(post.at(i) * ge, ho, s1[0]);
    }
    if (a.dx) P::store(static_cast<T *>(a.dx) + row * a.ldx, d, a.cols, t);
    if (a.dout) {
      float mo = 0.0f;
      if (a.post_norm) {
        sum1(s1);
        mo = s1[0] / (float)a.cols;
      }
      // e again from the fp32 t: d holds stream_scale t, which may be 0
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        const float hr = pr.at(i) * ir, ho = po.at(i) * io;
        const float tt = fmaf(ir, fmaf(pre.at(i), py.at(i), -hr * mr), pd.at(i));
        const float ge = g.at(i) * (a.branch_scale * tt);
        d[i] = a.post_norm ? io * fmaf(post.at(i), ge, -ho * mo) : ge;
      }
      P::store(static_cast<T *>(a.dout) + row * a.ldo, d, a.cols, t);
    }
    // The last row of a gate row whose rows all are this worker's.
    if (a.dgate && a.split == 1 && (row + 1 == a.rows || (row + 1) % a.group == 0)) {
      P::store(static_cast<T *>(a.dgate) + row / a.group * a.ldg, agate, a.cols, t);
#pragma unroll
      for (int i = 0; i < NE; ++i) agate[i] = 0.0f;
    }
    if constexpr (kAhead) {
      po = no;
      pr = nr;
      pd = nd;
      py = ny;
      g = ng;
    } else if (row + 1 < end) {
      load(po, pr, pd, py, g, row + 1);
    }
  }
  if (a.part_pre) P::store_f32(a.part_pre + w * a.cols, apre, a.cols, t);
  if (a.part_post) P::store_f32(a.part_post + w * a.cols, apost, a.cols, t);
  if (a.part_gate) P::store_f32(a.part_gate + w * a.cols, agate, a.cols, t);
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
  uint64_t row, end;
  if (!worker_rows(a, w, row, end)) return;
  // Partial rows are summed in memory, each column by one thread.
  float *parts[3] = {a.part_pre, a.part_post, a.part_gate};
  for (float *p : parts)
    if (p)
      for (uint32_t c = threadIdx.x; c < a.cols; c += kGenNT) p[w * a.cols + c] = 0.0f;
  for (; row < end; ++row) {
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
// dpost, 2 + g: dgate of gate row g (its `split` workers).  Four waves take a
// quarter of the rows each, eight loads in flight, then add in order.
template <class T>
__device__ __forceinline__ void finish(const BwppResNormArgs &a) {
  __shared__ float s[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t c = blockIdx.x * 64 + lane, which = blockIdx.y;
  const float *part = which == 0 ? a.part_pre : which == 1 ? a.part_post : a.part_gate;
  T *out = static_cast<T *>(which == 0 ? a.dpre : which == 1 ? a.dpost : a.dgate);
  if (!part || !out) return;
  uint32_t n = a.workers;
  if (which >= 2) {
    part += (uint64_t)(which - 2) * a.split * a.cols;
    out += (uint64_t)(which - 2) * a.ldg;
    n = a.split;
  }
  const uint32_t q = (n + 3) / 4, p0 = min(wave * q, n), p1 = min(p0 + q, n);
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
  if (wave == 0 && c < a.cols) out[c] = Elem<T>::of((s[0][lane] + s[1][lane]) + (s[2][lane] + s[3][lane]));
}

}  // namespace

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
  BWPP_RESNORM_GRAD(TN, T, 8, 1)                                                                               \
  BWPP_RESNORM_GRAD(TN, T, 8, 2)                                                                               \
  BWPP_RESNORM_GRAD(TN, T, 8, 4)                                                                               \
  BWPP_RESNORM_GRAD(TN, T, 8, 8)                                                                               \
  BWPP_RESNORM_GRAD(TN, T, 8, 16)                                                                              \
  extern "C" __global__ __launch_bounds__(kGenNT) void bwpp_resnorm_##TN##_any(const BwppResNormArgs a) {      \
    forward_any<T>(a);                                                                                         \
  }                                                                                                            \
  extern "C" __global__ __launch_bounds__(kGenNT) void bwpp_resnorm_grad_##TN##_any(const BwppResNormArgs a) { \
    gradient_any<T>(a);                                                                                        \
  }                                                                                                            \
  extern "C" __global__ __launch_bounds__(256) void bwpp_resnorm_finish_##TN(const BwppResNormArgs a) { finish<T>(a); }
BWPP_RESNORM_ALL(bf16, uint16_t)
BWPP_RESNORM_ALL(f32, float)
