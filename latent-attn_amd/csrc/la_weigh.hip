// The attention weight that cache rows get (la_weigh_kv):
//   w[s, p] += sum_{t, h} 2^(x[t, h, p] - lse[t, h]),  x = scale log2(e) (q_abs . c_t[p] + q_rope . RoPE(k_rope[p], p)),
// over the sequence's last tokens t (causal) and all heads h, lse the base-2
// log-sum-exp of a row of x. The weights are sums over many steps that rank rows
// against each other, so they and the scores are kept to fp32.
#include "la_draft.hpp"

namespace la {
namespace {

constexpr float kNoScore = -1e30f;
constexpr int kLatent = 1024;  // kv_lora_rank at most: 16 elements per lane

// One row's score against one query, by a wave: q (lane + 64 i) and the row's elements in the lanes.
__device__ inline float plain_score(const WeighProblem& p, const float (&q)[16], const float* qr, int s, int k, int lane) {
  const int half = p.dR / 2;
  const int64_t row = source_row(p.src, s, k) * p.src.row_elems, rk = source_rope_row(p.src, k) * half;
  float d = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (lane + 64 * i < p.dc) d += q[i] * load_any(p.src.kv, p.src.kv_dtype, row + lane + 64 * i);
  for (int i = lane; i < half; i += 64) {
    const float k0 = load_any(p.src.kv, p.src.kv_dtype, row + p.dc + i);
    const float k1 = load_any(p.src.kv, p.src.kv_dtype, row + p.dc + i + half);
    const float cs = p.src.cos[rk + i], sn = p.src.sin[rk + i];
    d += qr[i] * (k0 * cs - k1 * sn) + qr[i + half] * (k0 * sn + k1 * cs);
  }
  return wave_sum(d) * p.scale_log2;
}
__device__ inline void plain_query(const WeighProblem& p, int64_t item, int lane, float (&q)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) q[i] = lane + 64 * i < p.dc ? p.q_abs[item * p.dc + lane + 64 * i] : 0.f;
}

// The plain form, for any type and head shape: a workgroup of 4 waves per
// (token, head) for the log-sum-exps, then a wave per row that goes through
// all (token, head) again. Sums in a fixed order. Bound by the rows' and the
// queries' way from the L2.
__global__ __launch_bounds__(256) void plain_lse_kernel(WeighProblem p, int64_t first) {
  __shared__ float ml[4][2];
  const uint32_t item = (uint32_t)first + blockIdx.x;
  const int token = (int)(item / p.nh), s = token / p.tokens, j = token % p.tokens;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int keys = source_rows(p.src, s) - p.tokens + j + 1;
  float q[16], m = kNoScore, l = 0.f;
  plain_query(p, item, lane, q);
  for (int k = wave; k < keys; k += 4) {
    const float x = plain_score(p, q, p.q_rope + item * (int64_t)p.dR, s, k, lane), up = fmaxf(m, x);
    l = l * exp2f(m - up) + exp2f(x - up);
    m = up;
  }
  if (lane == 0) {
    ml[wave][0] = m;
    ml[wave][1] = l;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float top = kNoScore, total = 0.f;
    for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][0]);
    for (int w = 0; w < 4; ++w) total += ml[w][1] * exp2f(ml[w][0] - top);
    p.lse[item] = keys > 0 ? top + log2f(total) : INFINITY;  // no row gets anything of a token that sees none
  }
}
__global__ __launch_bounds__(256) void plain_weigh_kernel(WeighProblem p, int s, int64_t first) {
  const int lane = threadIdx.x & 63, L = source_rows(p.src, s);
  const int64_t k = (first + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (k >= L) return;
  float sum = 0.f;
  const int j0 = max((int)k - (L - p.tokens), 0);  // the first token that sees row k
  for (int64_t item = ((int64_t)s * p.tokens + j0) * p.nh; item < (int64_t)(s + 1) * p.tokens * p.nh; ++item) {
    float q[16];
    plain_query(p, item, lane, q);
    sum += exp2f(plain_score(p, q, p.q_rope + item * p.dR, s, (int)k, lane) - p.lse[item]);
  }
  const int64_t at = (p.src.offsets ? source_begin(p.src, s) : (int64_t)s * p.src.region) + k;
  if (lane == 0) p.weights[at] += sum;
}

}  // namespace

hipError_t launch_weigh_plain(const WeighProblem& p, hipStream_t stream) {
  const int64_t items = (int64_t)p.src.num_seqs * p.tokens * p.nh;
  if (items > INT32_MAX || p.dc > kLatent) return hipErrorInvalidValue;
  hipError_t e = in_grids(items, most_blocks(256), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL(plain_lse_kernel, dim3(blocks), dim3(256), 0, stream, p, first);
  });
  const int64_t most = p.src.offsets ? p.src.total_rows : p.src.region;
  for (int s = 0; s < p.src.num_seqs && e == hipSuccess; ++s)
    e = in_grids((most + 3) / 4, most_blocks(256), [&](int64_t first, unsigned blocks) {
      hipLaunchKernelGGL(plain_weigh_kernel, dim3(blocks), dim3(256), 0, stream, p, s, first);
    });
  return e;
}

}  // namespace la
