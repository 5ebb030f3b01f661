// Rules for the next token on rows of logits.  For a token v of the vocabulary
// and a row's history, of which the first `prompt` tokens were given and the
// rest written by the model (v written c times):
//   v in the history:  z = z > 0 ? z / repetition : z repetition
//   z = z - (frequency c + [c > 0] presence) + bias[v]
//   v forbidden by the mask (its bit 0): z = -inf
//
// Bound by HBM: a logit is read and written once.  A block takes a chunk of
// one row's columns, counts the row's history in LDS (bit 31: v was given, below
// it c; whole numbers, so the order of the additions does not matter) and then
// goes over its chunk, which it has fetched meanwhile.  256 rows of 131072, fp32,
// histories of up to 8192 tokens: 63 us, 4.4 TB/s (chunks of 8192 the same); 4 of
// 32000: 6.8, a launch and a chain of latencies.
//
// x, read once, goes past the caches at every size: never slower than 3 % (the noise of
// small calls), 16 % faster at best.  500 tokens of history a row, fp32, past them and
// through them, x in memory: 4 rows of 32000 5.9 and 5.8 us, 64 of 131072 12.9 and 13.6, 256
// of 32000 12.8 and 14.8, 256 of 131072 52.0 and 52.5; with the copy that writes x right
// before: 9.8 and 9.9, 23.4 and 23.6, 24.0 and 23.3, 92.6 and 93.8 (bf16 512 of 131072
// 132 and 139).
#pragma once

#include "common.h"
#include "rotary_math.h"
#include "../kargs.h"

using namespace bwpp;

namespace logits {

constexpr uint32_t kPer = 4;   // 4-element chunks a thread
constexpr uint32_t kPast = 8;  // tokens of the history on the way at once

template <class TX, class TY>
__device__ __forceinline__ void rules(const BwppLogitArgs &a) {
  using rotary_pos::Vec;
  extern __shared__ uint32_t seen[];
  const uint32_t row = blockIdx.x / a.chunks, c0 = blockIdx.x % a.chunks * a.chunk, NT = blockDim.x;
  const uint32_t nc = min(a.chunk, a.vocab - c0), n4 = nc / 4u;
  const TX *x = static_cast<const TX *>(a.x) + row * a.ldx + c0;
  TY *y = static_cast<TY *>(a.y) + row * a.ldy + c0;
  float v[kPer][4];  // on the way while the history is counted
#pragma unroll
  for (uint32_t j = 0; j < kPer; ++j)
    if (threadIdx.x + j * NT < n4) Vec<TX, 4>::load_once(x + 4u * (threadIdx.x + j * NT), v[j]);

  uint32_t n = 0;
  if (a.count) {
    const int32_t s0 = a.starts[row], s1 = a.starts[row + 1];
    const uint32_t b = s0 < 0 ? 0u : min((uint32_t)s0, a.history_len), e = s1 < 0 ? 0u : min((uint32_t)s1, a.history_len);
    n = e > b ? e - b : 0u;
    const int32_t *past = a.history + b;
    const int32_t p = a.prompt ? a.prompt[row] : 0;
    const uint32_t prompt = p < 0 ? 0u : (uint32_t)p;
    if (n) {  // uniform in the block
      for (uint32_t i = threadIdx.x; i < nc; i += NT) seen[i] = 0u;
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < n; i += kPast * NT) {
        uint32_t t[kPast];
#pragma unroll
        for (uint32_t j = 0; j < kPast; ++j) t[j] = i + j * NT < n ? (uint32_t)past[i + j * NT] - c0 : ~0u;
#pragma unroll
        for (uint32_t j = 0; j < kPast; ++j)
          if (t[j] < nc) {
            if (i + j * NT >= prompt) atomicAdd(&seen[t[j]], 1u);
            else atomicOr(&seen[t[j]], 0x80000000u);
          }
      }
      __syncthreads();
    }
  }
  const float rho = a.repetition ? a.repetition[row] : 1.0f;
  const float pres = a.presence ? a.presence[row] : 0.0f, freq = a.frequency ? a.frequency[row] : 0.0f;
  const float *bias = a.bias ? a.bias + row * a.ld_bias + c0 : nullptr;
  const uint32_t *mask = a.mask ? a.mask + row * a.ld_mask + c0 / 32u : nullptr;  // chunks are multiples of 32

  auto rule = [&](float z, uint32_t i, float b, uint32_t bits) {
    if (n) {
      const uint32_t w = seen[i];
      if (w) {
        if (a.repetition) z = z > 0.0f ? z / rho : z * rho;
        const uint32_t said = w & 0x7fffffffu;
        if (said) z -= freq * (float)said + pres;
      }
    }
    if (bias) z += b;
    return mask && !((bits >> (i & 31u)) & 1u) ? -INFINITY : z;
  };
#pragma unroll
  for (uint32_t j = 0; j < kPer; ++j) {
    const uint32_t i = threadIdx.x + j * NT;
    if (i >= n4) break;
    float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (bias) Vec<float, 4>::load(bias + 4u * i, b);
    const uint32_t bits = mask ? mask[i / 8u] : 0u;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) v[j][e] = rule(v[j][e], 4u * i + e, b[e], bits);
    Vec<TY, 4>::store(y + 4u * i, v[j]);
  }
  for (uint32_t i = 4u * n4 + threadIdx.x; i < nc; i += NT) {
    float w[1];
    Vec<TX, 1>::load_once(x + i, w);
    w[0] = rule(w[0], i, bias ? bias[i] : 0.0f, mask ? mask[i / 32u] : 0u);
    Vec<TY, 1>::store(y + i, w);
  }
}

}  // namespace logits

#define BWPP_RULES(NAME, TX, TY) \
  extern "C" __global__ __launch_bounds__(1024) void bwpp_logit_rules_##NAME(const BwppLogitArgs a) { logits::rules<TX, TY>(a); }
BWPP_RULES(f32, float, float)
BWPP_RULES(f32_bf16, float, uint16_t)
BWPP_RULES(bf16_f32, uint16_t, float)
BWPP_RULES(bf16, uint16_t, uint16_t)
