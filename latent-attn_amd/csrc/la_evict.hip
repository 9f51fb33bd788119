// Eviction (la_evict_kv): every sequence that is too long keeps its first and last
// rows and the heaviest ones between, in order and in place.
//
// Selection, one workgroup per sequence: the weights become keys that order as
// unsigned numbers, the k-th largest key is found 11 bits at a time from
// histograms in LDS (radix selection: three passes over the keys, which stay in
// registers up to 16,384 rows), and one pass in order keeps what is larger and as
// many of the equal ones as are left, earliest first, moving the weights on its
// way (position i goes to i or before, and a pass's writes follow its reads).
// Rows are counted in unsigned numbers: up to 2^31 - 1 of them, and as many asked for, the last step passes 2^31.
// Every wave has consecutive rows, so ranks are ballots and one sum over the waves.
//
// Movement: rows only move down, and the columns of a row are independent of
// one another. So a workgroup owns a stripe of columns of a sequence and goes
// through the kept rows in order, a tile of them read before any of it is
// written: no row is overwritten before its stripe is read, and no workgroup
// waits for another. A few sequences have too few stripes for that; their rows go
// through a copy, two launches over all compute units.
//
// What bounds it (bf16): 32 sequences of 8192 rows cut to 2048, 67 us in the two kernels: selection 18, five
// rounds of barriers over registers on 32 compute units; movement 49 for 147 MB from HBM, 3.0 TB/s (37 from
// the caches, where the same inputs come again and again). 1001 rows of one to 512: 20 us, latency.
#include "la_draft.hpp"

#include <algorithm>
#include <type_traits>

namespace la {
namespace {

constexpr int kItems = 16;  // rows of a lane at a time
constexpr int kBins = 2048;

// Largest first; NaN below everything, -0 as 0.
__device__ inline uint32_t key_of(float w) {
  if (w != w) return 0;
  const uint32_t u = u_of(w == 0.f ? 0.f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum of v over the waves before this one, and over all; one barrier (`sums` is used once).
template <int kW>
__device__ inline int wave_rank(int v, int* sums, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) sums[wave] = v;
  __syncthreads();
  const int mine = lane < kW ? sums[lane] : 0, end = wave_scan(mine);
  *total = __builtin_amdgcn_readlane(end, 63);
  return __builtin_amdgcn_readlane(end - mine, __builtin_amdgcn_readfirstlane(wave));
}

template <int kW>
__global__ __launch_bounds__(64 * kW) void evict_select_kernel(EvictProblem p, int64_t first_seq) {
  constexpr int kThreads = 64 * kW, kSegment = kItems * kThreads;
  __shared__ int hist[3][kBins];
  __shared__ int sums[5][kW];
  __shared__ int pick[3][2];
  __shared__ int moved;
  const int s = (int)first_seq + blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t begin = moved_begin(p.rows, s);
  const uint32_t L = (uint32_t)max(min(p.rows.lens[s], moved_room(p.rows, s)), 0), keep = (uint32_t)p.keep;
  float* const w = p.weights + begin;
  int32_t* const kept = p.kept + (int64_t)s * p.keep;
  if (L <= keep) {
    for (uint32_t i = tid; i < keep; i += kThreads) kept[i] = i < L ? (int32_t)i : -1;
    if (tid == 0) p.start[s] = p.keep;
    return;
  }
  uint32_t* const from = p.from + (int64_t)s * p.keep;
  const uint32_t lo = p.first, hi = L - p.last;  // the rows between
  int left = p.keep - p.first - p.last;     // of which so many stay
  const int segments = (int)((L + kSegment - 1) / kSegment);
  // of segment g a wave has 64 each(g) rows from at(g) on, 64 at a time
  auto each = [&](int g) { return (int)((min(L - g * (uint32_t)kSegment, (uint32_t)kSegment) + kThreads - 1) / kThreads); };
  auto at = [&](int g) { return g * (uint32_t)kSegment + wave * 64 * each(g) + lane; };
  float x[kItems];
  auto load = [&](int g) {
    const int n = each(g);
    const uint32_t i0 = at(g);
#pragma unroll
    for (int e = 0; e < kItems; ++e) x[e] = e < n && i0 + 64 * e < L ? w[i0 + 64 * e] : 0.f;
  };
  load(0);
  for (int i = tid; i < 3 * kBins; i += kThreads) hist[0][i] = 0;
  if (tid == 0) moved = p.keep;
  __syncthreads();
  // the left-th largest key between, and how many equal to it stay
  uint32_t prefix = left > 0 ? 0 : ~0u;  // (no key is as large: nothing between stays)
  if (left > 0) {
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int g = 0; g < segments; ++g) {
        if (segments > 1) load(g);
        const int n = each(g);
        const uint32_t i0 = at(g);
#pragma unroll
        for (int e = 0; e < kItems; ++e) {
          if (e >= n) break;
          const uint32_t i = i0 + 64 * e;
          const uint32_t k = key_of(x[e]);
          if (i >= lo && i < hi && (pass == 0 || k >> (shift + bits) == prefix >> (shift + bits)))
            atomicAdd(&hist[pass][k >> shift & ((1 << bits) - 1)], 1);
        }
      }
      __syncthreads();
      // this thread's bins, from the largest down
      constexpr int kEach = kBins / kThreads;
      int c[kEach], own = 0;
#pragma unroll
      for (int q = 0; q < kEach; ++q) own += c[q] = hist[pass][kBins - 1 - kEach * tid - q];
      const int in = wave_scan(own);
      int total;
      int more = wave_rank<kW>(__builtin_amdgcn_readlane(in, 63), sums[pass], &total) + in - own;
      if (more < left && left <= more + own) {
#pragma unroll
        for (int q = 0; q < kEach; ++q) {
          if (more < left && left <= more + c[q]) {
            pick[pass][0] = kBins - 1 - kEach * tid - q;
            pick[pass][1] = left - more;
          }
          more += c[q];
        }
      }
      __syncthreads();
      prefix |= (uint32_t)pick[pass][0] << shift;
      left = pick[pass][1];
    }
  }
  // in order: what is larger, and the first `left` of the equal ones
  const uint64_t before = (1ull << lane) - 1;
  int done = 0, equal = 0, moves = p.keep;
  for (int g = 0; g < segments; ++g) {
    if (segments > 1) {
      load(g);
      __syncthreads();  // the sums of the segment before are read
    }
    const int n = each(g);
    const uint32_t i0 = at(g);
    int same = 0, total;
#pragma unroll
    for (int e = 0; e < kItems; ++e) {
      if (e >= n) break;
      const uint32_t i = i0 + 64 * e;
      same += __popcll(__builtin_amdgcn_ballot_w64(i >= lo && i < hi && key_of(x[e]) == prefix));
    }
    int rank = equal + wave_rank<kW>(same, sums[3], &total);
    equal += total;
    uint32_t stays = 0;
    int count = 0;
#pragma unroll
    for (int e = 0; e < kItems; ++e) {
      if (e >= n) break;
      const uint32_t i = i0 + 64 * e;
      const uint32_t k = key_of(x[e]);
      const bool between = i >= lo && i < hi, is = between && k == prefix;
      const uint64_t all = __builtin_amdgcn_ballot_w64(is);
      const bool stay = i < L && (!between || k > prefix || (is && rank + __popcll(all & before) < left));
      rank += __popcll(all);
      stays |= (uint32_t)stay << e;
      count += __popcll(__builtin_amdgcn_ballot_w64(stay));
    }
    int to = done + wave_rank<kW>(count, sums[4], &total);  // (its barrier: every weight of the segment is read)
    done += total;
#pragma unroll
    for (int e = 0; e < kItems; ++e) {
      if (e >= n) break;
      const bool stay = stays >> e & 1;
      const uint64_t all = __builtin_amdgcn_ballot_w64(stay);
      const uint32_t i = i0 + 64 * e, mine = to + __popcll(all & before);
      to += __popcll(all);
      if (stay && mine < keep) {
        kept[mine] = (int32_t)i;
        from[mine] = (uint32_t)moved_index(p.rows, s, begin, (int)i);
        if (mine != i) {
          w[mine] = x[e];
          moves = min(moves, (int)mine);
        }
      }
    }
  }
  // Weights that another sequence moves meanwhile (offsets that overlap) are other ones at every look: the rows that
  // stay are then not as many as they should be, and every entry still has to name a row.
  for (uint32_t i = done + tid; i < keep; i += kThreads) {
    kept[i] = (int32_t)i;
    from[i] = (uint32_t)moved_index(p.rows, s, begin, (int)i);
  }
  if (moves < p.keep) atomicMin(&moved, moves);
  __syncthreads();
  for (uint32_t i = keep + tid; i < L; i += kThreads) w[i] = 0.f;
  if (tid == 0) {
    p.start[s] = moved;
    p.rows.lens[s] = p.keep;
  }
}

// kLanes units of U per row and workgroup, kRows rows at a time, kDeep of these in
// flight and as many more on their way behind them.
constexpr int kMoveThreads = 256, kLanes = 8, kRows = kMoveThreads / kLanes, kDeep = 8;
template <typename U>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictProblem p, int stripes, int64_t first) {
  const int64_t item = first + blockIdx.x;
  const int s = (int)(item / stripes), units = (int)(p.rows.row_bytes / sizeof(U));
  const int column = (int)(item % stripes) * kLanes + threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const bool in = column < units;
  const int64_t begin = moved_begin(p.rows, s);
  const uint32_t* const from = p.from + (int64_t)s * p.keep;
  const U* const base = reinterpret_cast<const U*>(p.rows.kv) + min(column, units - 1);
  const uint32_t start = p.start[s], keep = (uint32_t)p.keep;
  if (start >= keep) return;
  typedef typename std::conditional<(sizeof(U) < 4), uint32_t, U>::type H;  // (a register each)
  auto load = [&](uint32_t i0, H(&v)[kDeep]) {  // (rows past the last: the last again)
#pragma unroll
    for (int k = 0; k < kDeep; ++k) v[k] = base[(int64_t)from[min(i0 + k * kRows + row, keep - 1)] * units];
  };
  auto store = [&](uint32_t i0, H(&v)[kDeep]) {
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const uint32_t i = i0 + k * kRows + row;
      if (in && i < keep) reinterpret_cast<U*>(moved_row(p.rows, s, begin, (int)i))[column] = (U)v[k];
    }
  };
  // everyone's rows of a tile are read before anyone writes it
  auto read = [](H(&v)[kDeep]) {
#pragma unroll
    for (int k = 0; k < kDeep; ++k) asm volatile("" : "+v"(v[k]));
    lds_barrier();
  };
  constexpr uint32_t kTile = kRows * kDeep;
  H a[kDeep], b[kDeep];
  load(start, a);
  for (uint32_t i0 = start; i0 < keep; i0 += 2 * kTile) {
    load(min(i0 + kTile, keep - 1), b);
    read(a);
    store(i0, a);
    if (i0 + kTile >= keep) break;
    load(min(i0 + 2 * kTile, keep - 1), a);
    read(b);
    store(i0 + kTile, b);
  }
}

// Unit by unit, to the copy (kOut) and back.
template <typename U, bool kOut>
__global__ __launch_bounds__(256) void evict_copy_kernel(EvictProblem p, int blocks_per) {
  const int s = blockIdx.x / blocks_per, b = blockIdx.x % blocks_per, units = (int)(p.rows.row_bytes / sizeof(U));
  const int start = p.start[s];
  const int64_t begin = moved_begin(p.rows, s), all = (int64_t)(p.keep - start) * units;
  U* const copy = reinterpret_cast<U*>(p.staged) + ((int64_t)s * p.keep + start) * units;
  const uint32_t* const from = p.from + (int64_t)s * p.keep;
  for (int64_t u = (int64_t)b * 256 + threadIdx.x; u < all; u += (int64_t)blocks_per * 256) {
    const int i = start + (int)(u / units), c = (int)(u % units);
    if constexpr (kOut) copy[u] = (reinterpret_cast<const U*>(p.rows.kv) + (int64_t)from[i] * units)[c];
    else reinterpret_cast<U*>(moved_row(p.rows, s, begin, i))[c] = copy[u];
  }
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename U>
hipError_t move_t(const EvictProblem& p, hipStream_t stream) {
  const int64_t units = p.rows.row_bytes / sizeof(U);
  if (p.staged) {
    const int64_t each = (p.keep * units + 1023) / 1024, most = std::max<int64_t>(4096 / p.rows.num_seqs, 1);
    const int blocks = (int)std::max<int64_t>(std::min(each, most), 1);
    hipLaunchKernelGGL((evict_copy_kernel<U, true>), dim3((unsigned)(p.rows.num_seqs * blocks)), dim3(256), 0, stream, p, blocks);
    hipLaunchKernelGGL((evict_copy_kernel<U, false>), dim3((unsigned)(p.rows.num_seqs * blocks)), dim3(256), 0, stream, p, blocks);
    return hipGetLastError();
  }
  const int stripes = (int)((units + kLanes - 1) / kLanes);
  return in_grids((int64_t)p.rows.num_seqs * stripes, most_blocks(kMoveThreads), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL(evict_move_kernel<U>, dim3(blocks), dim3(kMoveThreads), 0, stream, p, stripes, first);
  });
}

}  // namespace

// Two launches over all compute units against stripes, whose time goes by the rows kept. A call over 576 bf16
// elements a row (9 stripes, so up to 14 sequences take the copy), us, stripes / copy:
//   1 sequence, 1001 rows to 512 17.2 / 19.3, 8192 to 512 23.8 / 25.6, to 2048 30.3 / 26.5, 32,768 to 512 54.5 / 56.5,
//     to 2048 62.1 / 57.8, to 16,384 123 / 65.4
//   4 of 1001 to 512 17.7 / 20.0, 8192 to 2048 31.8 / 29.7, 32,768 to 16,384 152 / 101
//   13 of 1001 to 512 18.6 / 22.6, 8192 to 2048 35.6 / 42.5; 16 of 8192 to 2048 38.0 / 49.4; 32 58.3 / 73.5
// The lengths are on the device and most of a copy's gain is where much is kept: a few us lost below, 50 gained above.
bool evict_staged(const EvictProblem& p, int ncu) {
  const int unit = moved_unit(p.rows);
  return p.rows.num_seqs * ((p.rows.row_bytes / unit + kLanes - 1) / kLanes) < ncu / 2;
}

hipError_t launch_evict(const EvictProblem& p, hipStream_t stream) {
  // (short sequences: fewer waves meet sooner at every barrier)
  const bool few = !p.rows.offsets && p.rows.region <= 4 * 64 * kItems;
  const hipError_t e = in_grids(p.rows.num_seqs, most_blocks(1024), [&](int64_t first, unsigned blocks) {
    if (few) hipLaunchKernelGGL(evict_select_kernel<4>, dim3(blocks), dim3(256), 0, stream, p, first);
    else hipLaunchKernelGGL(evict_select_kernel<16>, dim3(blocks), dim3(1024), 0, stream, p, first);
  });
  if (e != hipSuccess || p.keep == 0 || !p.from) return e;
  switch (moved_unit(p.rows)) {
    case 16: return move_t<u32x4>(p, stream);
    case 8: return move_t<uint64_t>(p, stream);
    case 4: return move_t<uint32_t>(p, stream);
    case 2: return move_t<uint16_t>(p, stream);
    default: return move_t<uint8_t>(p, stream);
  }
}

}  // namespace la
