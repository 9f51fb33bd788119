// Eviction (la_evict_kv): every sequence that is too long keeps its first and last
// rows and the heaviest ones between, in order and in place.
//
// Selection, one workgroup per sequence: the weights become keys that order as
// unsigned numbers, the k-th largest key is found 8 bits at a time from
// histograms in LDS (radix selection), and one pass in order keeps what is
// larger and as many of the equal ones as are left, earliest first, moving the
// weights on its way (position i goes to i or before, and a pass's writes follow
// its reads).
//
// Movement: rows only move down, and the columns of a row are independent of
// one another. So a workgroup owns a stripe of columns of a sequence and goes
// through the kept rows in order, a tile of them read before any of it is
// written: no row is overwritten before its stripe is read, and no workgroup
// waits for another.
#include "la_draft.hpp"

namespace la {
namespace {

constexpr int kSelectThreads = 1024;

// Largest first; NaN below everything, -0 as 0.
__device__ inline uint32_t key_of(float w) {
  if (w != w) return 0;
  const uint32_t u = u_of(w == 0.f ? 0.f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum over the workgroup's threads in order, and the total.
__device__ inline int block_scan(int v, int* sums, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int in = wave_scan(v);
  __syncthreads();
  if (lane == 63) sums[wave] = in;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kSelectThreads / 64; ++w) {
    before += w < wave ? sums[w] : 0;
    all += sums[w];
  }
  *total = all;
  return before + in - v;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(EvictProblem p, int64_t first_seq) {
  __shared__ int hist[256];
  __shared__ int sums[kSelectThreads / 64];
  __shared__ uint32_t pick[2];
  const int s = (int)first_seq + blockIdx.x;
  const int64_t begin = moved_begin(p.rows, s);
  const int L = max(min(p.rows.lens[s], moved_room(p.rows, s)), 0);
  float* const w = p.weights + begin;
  int32_t* const kept = p.kept + (int64_t)s * p.keep;
  if (L <= p.keep) {
    for (int i = threadIdx.x; i < p.keep; i += kSelectThreads) kept[i] = i < L ? i : -1;
    if (threadIdx.x == 0) p.start[s] = p.keep;
    return;
  }
  const int lo = p.first, hi = L - p.last;  // the rows between
  int left = p.keep - p.first - p.last;     // of which so many stay
  // the left-th largest key between, and how many equal to it stay
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    for (int i = lo + threadIdx.x; i < hi; i += kSelectThreads) {
      const uint32_t k = key_of(w[i]);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int n = left, b = 255;
      while (b > 0 && hist[b] < n) n -= hist[b--];
      pick[0] = (uint32_t)b;
      pick[1] = (uint32_t)n;
    }
    __syncthreads();
    prefix |= pick[0] << shift;
    left = (int)pick[1];
    __syncthreads();
  }
  // in order: what is larger, the first `left` of the equal ones (none where no row between stays)
  if (p.keep == p.first + p.last) prefix = ~0u, left = 0;
  int at = 0, equal = 0;
  for (int i0 = 0; i0 < L; i0 += kSelectThreads) {
    const int i = i0 + threadIdx.x;
    const float x = i < L ? w[i] : 0.f;
    const uint32_t k = key_of(x);
    const bool between = i >= lo && i < hi, same = between && k == prefix;
    int total;
    const int rank = equal + block_scan(same ? 1 : 0, sums, &total);
    equal += total;
    const bool stays = i < L && (!between || (same ? rank < left : k > prefix));
    const int to = at + block_scan(stays ? 1 : 0, sums, &total);  // (its barriers: every weight of the pass is read)
    if (stays) {
      kept[to] = i;
      if (to != i) w[to] = x;
    }
    at += total;
  }
  __syncthreads();
  for (int i = p.keep + threadIdx.x; i < L; i += kSelectThreads) w[i] = 0.f;
  // the first position that gets another row
  if (threadIdx.x == 0) pick[0] = (uint32_t)p.keep;
  __syncthreads();
  for (int i = threadIdx.x; i < p.keep; i += kSelectThreads)
    if (kept[i] != i) {
      atomicMin(&pick[0], (uint32_t)i);
      break;
    }
  __syncthreads();
  if (threadIdx.x == 0) {
    p.start[s] = (int)pick[0];
    p.rows.lens[s] = p.keep;
  }
}

// kRows rows of kLanes units of kU bytes at a time, kDeep of these in flight.
constexpr int kMoveThreads = 256;
template <typename U, int kLanes>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictProblem p, int stripes, int64_t first) {
  constexpr int kRows = kMoveThreads / kLanes, kDeep = 8;
  const int64_t item = first + blockIdx.x;
  const int s = (int)(item / stripes), column = (int)(item % stripes) * kLanes + threadIdx.x % kLanes;
  const int row = threadIdx.x / kLanes;
  const bool in = column < (int)(p.rows.row_bytes / sizeof(U));
  const int64_t begin = moved_begin(p.rows, s);
  const int32_t* const kept = p.kept + (int64_t)s * p.keep;
  for (int i0 = p.start[s]; i0 < p.keep; i0 += kRows * kDeep) {
    U v[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int i = i0 + k * kRows + row;
      if (in && i < p.keep) v[k] = reinterpret_cast<const U*>(moved_row(p.rows, s, begin, kept[i]))[column];
    }
    rows_read();
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int i = i0 + k * kRows + row;
      if (in && i < p.keep) reinterpret_cast<U*>(moved_row(p.rows, s, begin, i))[column] = v[k];
    }
  }
}

struct alignas(16) Unit16 {
  uint32_t x[4];
};

template <typename U>
hipError_t move_t(const EvictProblem& p, hipStream_t stream) {
  constexpr int kLanes = 8;
  const int stripes = (int)((p.rows.row_bytes / sizeof(U) + kLanes - 1) / kLanes);
  return in_grids((int64_t)p.rows.num_seqs * stripes, most_blocks(kMoveThreads), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL((evict_move_kernel<U, kLanes>), dim3(blocks), dim3(kMoveThreads), 0, stream, p, stripes, first);
  });
}

}  // namespace

hipError_t launch_evict(const EvictProblem& p, hipStream_t stream) {
  const hipError_t e = in_grids(p.rows.num_seqs, most_blocks(kSelectThreads), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL(evict_select_kernel, dim3(blocks), dim3(kSelectThreads), 0, stream, p, first);
  });
  if (e != hipSuccess) return e;
  switch (moved_unit(p.rows)) {
    case 16: return move_t<Unit16>(p, stream);
    case 8: return move_t<uint64_t>(p, stream);
    case 4: return move_t<uint32_t>(p, stream);
    case 2: return move_t<uint16_t>(p, stream);
    default: return move_t<uint8_t>(p, stream);
  }
}

}  // namespace la
