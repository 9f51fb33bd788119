// Joins partial attention results of the same query rows: out = sum_i 2^(e_i - M) o_i / sum_i 2^(e_i - M),
// e_i the base-2 log-sum-exp of part i and M the largest. Parts are the key
// splits of prompt_kernel and whole decode steps, whose log-sum-exps are
// those of their partial slots.
#include "la_prompt.hpp"

namespace la {
namespace {

__device__ inline float max32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ inline float sum32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Log-sum-exp of query row `row` of a decode step over its partial slots, by 32 lanes.
__device__ inline float step_lse(const DecodeProblem& p, int64_t row, int l32) {
  const int s = (int)(row / p.Hq), hq = (int)(row % p.Hq);
  int64_t lo, hi;
  const int len = seq_in_plan(p, s, &lo, &hi);
  if (hi <= lo) return -INFINITY;
  const int64_t cf = lo / len, cl = (hi - 1) / len;
  float m = -INFINITY;
  for (int64_t c = cf + l32; c <= cl; c += 32) m = fmaxf(m, p.part_lse[slot_of(p, c, s) * p.Hq + hq]);
  m = max32(m);  // (maxima pass over NaN, the sum below does not)
  float l = 0.f;
  for (int64_t c = cf + l32; c <= cl; c += 32) {
    const float e = p.part_lse[slot_of(p, c, s) * p.Hq + hq];
    l += e == -INFINITY ? 0.f : exp2f(e - m);
  }
  l = sum32(l);
  return l == 0.f ? -INFINITY : m + log2f(l);
}

// For parts that no merge can take along: key splits of a prompt, and decode
// steps of the VALU or fp32 kernels. 32 lanes per query row, four values each at
// a time where rows are whole vectors; bound by latency, then by the parts'
// bytes (1024 tokens x 16 heads x 3 parts 7.5 us, 25 MB). The decode results go
// out before the log-sum-exps are known: those take several dependent loads,
// which are most of the kernel's time.
template <bool kVec>
__global__ __launch_bounds__(256) void join_kernel(JoinProblem p, int64_t block0) {
  const int64_t row = (block0 + blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int l32 = threadIdx.x & 31;
  if (row >= p.rows) return;
  constexpr int kN = kVec ? 4 : 1;
  struct Part {
    float v[kN];
  };
  auto load = [](const float* o) {
    Part r;
    if constexpr (kVec) __builtin_memcpy(r.v, __builtin_assume_aligned(o, 16), 16);
    else r.v[0] = *o;
    return r;
  };
  Part first[2] = {};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (p.step[i].num_seqs > 0 && l32 * kN < p.dv) first[i] = load(p.step_out[i] + row * p.dv + l32 * kN);
  // lane i holds part i's weight
  const float e = l32 < p.splits ? p.part_lse[(int64_t)l32 * p.rows + row] : -INFINITY;
  float es[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (p.step[i].num_seqs > 0) es[i] = step_lse(p.step[i], row, l32);
  const float m = fmaxf(max32(e), fmaxf(es[0], es[1]));
  // rows that see nothing have no part with a weight; a NaN stays one
  const auto weight = [&](float x) { return x == -INFINITY ? 0.f : exp2f(x - m); };
  const float w = weight(e), ws[2] = {weight(es[0]), weight(es[1])};
  const float total = sum32(w) + ws[0] + ws[1];
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int base = threadIdx.x & 32;
  for (int d = l32 * kN; d < p.dv; d += 32 * kN) {
    float acc[kN] = {};
    auto add = [&](float f, const Part& o) {
#pragma unroll
      for (int k = 0; k < kN; ++k) acc[k] += f == 0.f ? 0.f : f * o.v[k];  // (a part without weight may hold anything)
    };
#pragma unroll 4
    for (int i = 0; i < p.splits; ++i)
      add(__shfl(w, base + i, 64), load(p.part_o + ((int64_t)i * p.rows + row) * p.dv + d));
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (p.step[i].num_seqs > 0) add(ws[i], d == l32 * kN ? first[i] : load(p.step_out[i] + row * p.dv + d));
    const int64_t at = row * p.dv + d;
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      const float v = acc[k] * inv;
      if (p.out_dtype == LA_DTYPE_F32) static_cast<float*>(p.out)[at + k] = v;
      else if (p.out_dtype == LA_DTYPE_BF16) static_cast<__bf16*>(p.out)[at + k] = (__bf16)v;
      else static_cast<_Float16*>(p.out)[at + k] = (_Float16)v;
    }
  }
}

}  // namespace

hipError_t launch_join(const JoinProblem& p, hipStream_t stream) {
  if (p.splits > kJoinSplits) return hipErrorInvalidValue;
  const auto k = p.dv % 4 == 0 ? join_kernel<true> : join_kernel<false>;
  return in_grids((p.rows + 7) / 8, most_blocks(256), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL(k, dim3(blocks), dim3(256), 0, stream, p, first);
  });
}

}  // namespace la
