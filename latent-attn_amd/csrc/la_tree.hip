// Trees of drafted tokens: what the attention over them takes (la_mla_decode_tree), its
// plain form, and the rows of an accepted path (la_accept_kv).
//
// Node j of a sequence's n <= 64 nodes has a parent before it or none. With
// A(j) = {j} and its ancestors as the bits of a word, A(j) = bit j | A(parent(j)): pointer
// doubling over the lanes of one wave finds all of them in six steps. depth(j) =
// |A(j)| - 1, and node j (query and key alike) is at position L - n + depth(j).
#include "la_draft.hpp"

namespace la {
namespace {

constexpr float kNoScore = -3.402823466e38f;  // no finite score is below

__device__ inline uint64_t shfl64(uint64_t v, int lane) {
  const uint32_t lo = __shfl((int)(uint32_t)v, lane, 64), hi = __shfl((int)(uint32_t)(v >> 32), lane, 64);
  return (uint64_t)hi << 32 | lo;
}
// A(lane) of sequence s's tree, by all lanes of a wave (0 past the nodes).
__device__ inline uint64_t tree_seen(const int32_t* parents, int s, int n) {
  const int lane = threadIdx.x & 63;
  int up = lane < n ? parents[(int64_t)s * n + lane] : -1;
  if (up < 0 || up >= lane) up = -1;
  uint64_t seen = lane < n ? 1ull << lane : 0;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const uint64_t more = shfl64(seen, up < 0 ? lane : up);
    const int next = __shfl(up, up < 0 ? lane : up, 64);
    if (up >= 0) {
      seen |= more;
      up = next;
    }
  }
  return seen;
}

// Rows of sequence s that its tree's attention reads.
__device__ inline int tree_rows(const TreeQueries& p, int s) {
  const int rows = source_rows(p.src, s);
  return rows < p.q.per_seq ? 0 : rows;
}
// The spans' plan (kSpans) of one wave. Either the tiles of all sequences are divided
// evenly, or every sequence starts a chunk of its own, at the fewest tiles a chunk that
// suffice. A chunk over several sequences pays kSegment tiles for each after the first
// (a segment's fixed part: its queries, its first tiles' way, its partial rows), own
// chunks for the shorter last ones: the smaller estimate of the longest chunk is taken.
// (16 trees of 16 behind 500 to 6000 rows, 128 heads, 16 chunks: own chunks 404 us a call, even
// ones 328. With 4, 8, 16 or 32 tiles for kSegment calls differ where it decides: 12 trees of 8 behind 200 to
// 9000 rows, 128 heads 163, 162, 153, 154; 20 of 16 behind 500 to 8000, 64 heads 231, 231, 231, 240; 16 of 16 and 4 of 64 the same.)
constexpr int kSegment = 8;
__device__ inline void plan_spans(const TreeQueries& p) {
  const int lane = wave_lane(), seqs = p.q.num_seqs;
  // 2^24 tiles: more than the memory holds; their sums stay below 2^31 (malformed offsets may overlap)
  auto tiles = [&](int s) { return s < seqs ? (int)min(((uint32_t)tree_rows(p, s) + kSpanRows - 1) / kSpanRows, 1u << 24) : 0; };
  constexpr int kHeld = 4;  // of the first 256 sequences, in registers
  int held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = tiles(lane + 64 * i);
  int64_t sum = 0;
  int have = 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) sum += held[i], have += held[i] > 0;
#pragma unroll 4
  for (int s = lane + 64 * kHeld; s < seqs; s += 64) {
    const int n = tiles(s);
    sum += n, have += n > 0;
  }
  // (in two parts: a lane's below 2^40 and so the 64 sums below 2^30)
  const int64_t total = (int64_t)wave_sum_i((int)min(sum >> 16, (int64_t)1 << 24)) * 65536 + wave_sum_i((int)(sum & 0xFFFF));
  const int filled = wave_sum_i(have);
  constexpr int kMost = kMaxChunkRows / kSpanRows;
  const int even = (int)min(max((total + p.chunks - 1) / p.chunks, (int64_t)p.shortest), (int64_t)kMost);
  int len = even;
  bool own = false;
  if (filled <= p.chunks) {
    auto fits = [&](int n) {
      int64_t count = 0;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) count += pieces(held[i], n);
      for (int s = lane + 64 * kHeld; s < seqs; s += 64) count += pieces(tiles(s), n);
      return wave_sum_i((int)min(count, (int64_t)1 << 24)) <= p.chunks;
    };
    int lo = even, hi = min(even + kSegment * ((filled - 1 + p.chunks - 1) / p.chunks), kMost);
    own = fits(hi);
    while (own && lo < hi) {
      const int mid = (lo + hi) / 2;
      if (fits(mid)) hi = mid;
      else lo = mid + 1;
    }
    if (own) len = hi;
  }
  len = min((len + p.step - 1) / p.step * p.step, kMost);
  int32_t* const first = p.lens + seqs;
  const int64_t limit = (int64_t)p.chunks * len;
  int64_t at = 0;
  for (int s0 = 0; s0 < seqs; s0 += 64) {
    int n = tiles(s0 + lane);
    if (own) n = pieces(n, len) * len;
    const int end = wave_scan(n);
    if (s0 + lane < seqs) first[s0 + lane] = (int)min(at + end - n, limit);
    at += __builtin_amdgcn_readlane(end, 63);
  }
  if (lane == 0) {
    first[seqs] = (int)min(at, limit);
    first[seqs + 1] = len;
  }
}

// As tokens_kernel: kElems elements of a token's nope queries, and as many pairs of
// rope ones, per workgroup (x: token, y: share), kN at a time; the first also
// writes what the tree's kernels take of its node.
constexpr int kElems = 2048;
template <int kN>
__device__ inline void load_n(const void* base, int dtype, int64_t i, float (&x)[kN]) {
  if constexpr (kN == 4) load_q4(base, dtype, i, x);
  else x[0] = load_any(base, dtype, i);
}
template <int kN>
__global__ __launch_bounds__(256) void tree_queries_kernel(TreeQueries p, int64_t token0) {
  const int64_t token = token0 + blockIdx.x;
  const int n = p.q.per_seq, s = (int)(token / n), j = (int)(token % n);
  const int L = tree_rows(p, s), half = p.dR / 2;
  const uint64_t seen = shfl64(tree_seen(p.parents, s, n), j);
  const int at = max(L - n + __popcll(seen) - 1, 0);
  const int64_t pos = source_rope_row(p.src, at);
  const float *const cos = p.src.cos + pos * half, *const sin = p.src.sin + pos * half;
  if (blockIdx.y == 0) {
    for (int i = threadIdx.x; i < half; i += 256) {
      p.cos[token * half + i] = cos[i];
      p.sin[token * half + i] = sin[i];
    }
    if (threadIdx.x == 0) {
      p.seen[token] = seen;
      if (p.pos) p.pos[token] = at;
      if (j == 0) p.lens[s] = L;
    }
    if (token == 0 && p.chunks > 0 && threadIdx.x >= 192) plan_spans(p);
  }
  const int first = blockIdx.y * kElems + kN * threadIdx.x, last = (blockIdx.y + 1) * kElems;
  if (p.q_nope)
    for (int i = first; i < min(last, p.nh * p.dn); i += kN * 256) {
      const int h = i / p.dn, d = i - h * p.dn;
      float x[kN];
      load_n<kN>(p.q.q_nope, p.q.dtype, token * p.q.nope_stride + h * p.q.nope_head + d, x);
#pragma unroll
      for (int e = 0; e < kN; ++e) p.q_nope[token * p.nh * p.dn + i + e] = x[e];
    }
  if (p.q_rope)
    for (int i = first; i < min(last, p.nh * half); i += kN * 256) {
      const int h = i / half, d = i - h * half;
      const int64_t from = token * p.q.rope_stride + h * p.q.rope_head + d;
      float a[kN], b[kN];
      load_n<kN>(p.q.q_rope, p.q.dtype, from, a);
      load_n<kN>(p.q.q_rope, p.q.dtype, from + half, b);
      float* const to = p.q_rope + (token * p.nh + h) * p.dR + d;
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float c = p.q.rotate ? cos[d + e] : 1.f, sn = p.q.rotate ? sin[d + e] : 0.f;
        to[e] = p.q.rotate ? a[e] * c - b[e] * sn : a[e];
        to[half + e] = p.q.rotate ? a[e] * sn + b[e] * c : b[e];
      }
    }
}

// The plain form: one workgroup of 4 waves per (token, head), from number
// first on; wave w takes rows w, w + 4, ... with a running maximum of its own,
// lanes share a row's elements, the waves' sums are joined and projected.
// Everything fp32. It is there for shapes and types that the matrix cores'
// kernels do not take; bound by the rows' way from the L2, once per head.
constexpr int kLatent = 1024;  // kv_lora_rank at most: 16 elements per lane
__global__ __launch_bounds__(256) void plain_tree_kernel(PlainTree p, int64_t first) {
  __shared__ float acc_l[4][kLatent];
  __shared__ float ml[4][2];
  const uint32_t item = (uint32_t)first + blockIdx.x;  // (tokens x heads stay below 2^31)
  const int64_t token = item / p.nh;
  const int h = (int)(item % p.nh);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int s = (int)(token / p.nodes), L = source_rows(p.src, s), before = L - p.nodes, half = p.dR / 2;
  const uint64_t seen = p.seen[token];
  const float *const qa = p.q_abs + item * (int64_t)p.dc, *const qr = p.q_rope + item * (int64_t)p.dR;
  float q[16], acc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    q[i] = lane + 64 * i < p.dc ? qa[lane + 64 * i] : 0.f;
    acc[i] = 0.f;
  }
  float m = kNoScore, l = 0.f;
  for (int64_t k64 = wave; k64 < L; k64 += 4) {  // (up to 2^31 - 1 rows)
    const int k = (int)k64;
    int64_t at = k;
    if (k >= before) {
      if (!(seen >> (k - before) & 1)) continue;
      at = before + __popcll(p.seen[(int64_t)s * p.nodes + k - before]) - 1;
    }
    const int64_t row = source_row(p.src, s, k) * p.src.row_elems, rk = source_rope_row(p.src, at) * half;
    float c[16], d = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      c[i] = lane + 64 * i < p.dc ? load_any(p.src.kv, p.src.kv_dtype, row + lane + 64 * i) : 0.f;
      d += q[i] * c[i];
    }
    for (int i = lane; i < half; i += 64) {
      const float k0 = load_any(p.src.kv, p.src.kv_dtype, row + p.dc + i);
      const float k1 = load_any(p.src.kv, p.src.kv_dtype, row + p.dc + i + half);
      const float cs = p.src.cos[rk + i], sn = p.src.sin[rk + i];
      d += qr[i] * (k0 * cs - k1 * sn) + qr[i + half] * (k0 * sn + k1 * cs);
    }
    const float x = scaled_score(wave_sum(d), p.scale_log2);
    const float up = fmaxf(m, x), a = exp2f(m - up), w = exp2f(x - up);
    m = up;
    l = l * a + w;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = acc[i] * a + w * c[i];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (lane + 64 * i < p.dc) acc_l[wave][lane + 64 * i] = acc[i];
  if (lane == 0) {
    ml[wave][0] = m;
    ml[wave][1] = l;
  }
  __syncthreads();
  float top = kNoScore, total = 0.f, f[4];
  for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][0]);
  for (int w = 0; w < 4; ++w) {
    f[w] = exp2f(ml[w][0] - top);
    total += f[w] * ml[w][1];
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  for (int i = threadIdx.x; i < p.dc; i += 256)
    acc_l[0][i] = (f[0] * acc_l[0][i] + f[1] * acc_l[1][i] + f[2] * acc_l[2][i] + f[3] * acc_l[3][i]) * inv;
  __syncthreads();
  for (int v = wave; v < p.dv; v += 4) {
    const int64_t w = ((int64_t)h * p.dv + v) * p.dc;
    float d = 0.f;
    for (int i = lane; i < p.dc; i += 64) d += acc_l[0][i] * load_any(p.W_UV, p.wuv_dtype, w + i);
    d = L > 0 ? wave_sum(d) : 0.f;
    if (lane == 0) {
      const int64_t at = item * (int64_t)p.dv + v;
      if (p.out_dtype == LA_DTYPE_F32) static_cast<float*>(p.out)[at] = d;
      else if (p.out_dtype == LA_DTYPE_BF16) static_cast<__bf16*>(p.out)[at] = (__bf16)d;
      else static_cast<_Float16*>(p.out)[at] = (_Float16)d;
    }
  }
}

// The rows of an accepted path. A workgroup has a sequence: it takes kAcceptPieces
// units of kU bytes per thread at a time, all read before any is written (a
// path's rows move down over rows that may be on it), columns of the rows being
// independent of one another. 16-bit rows of 576 elements and 64 nodes at most
// are one such step, so the kernel is three dependent loads (length, path,
// row) and the stores: latency is all there is (64 trees of 25 4.3 us, one of 64 3.5).
constexpr int kAcceptThreads = 1024, kAcceptPieces = 5;
template <typename U>
__global__ __launch_bounds__(kAcceptThreads) void accept_kernel(AcceptProblem p, int64_t first) {
  __shared__ int32_t path[kTreeNodes];
  __shared__ int count;
  const int s = (int)first + blockIdx.x, n = p.nodes;
  const int L = p.rows.lens[s];
  const int64_t begin = moved_begin(p.rows, s);
  if (L < n || L > moved_room(p.rows, s)) return;
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const int node = lane < n ? p.path[(int64_t)s * n + lane] : -1, last = __shfl_up(node, 1, 64);
    const uint64_t ends = __builtin_amdgcn_ballot_w64(node < 0 || node >= n || (lane > 0 && node <= last));
    path[lane] = node;
    if (lane == 0) count = ends ? __builtin_ctzll(ends) : 64;
  }
  __syncthreads();
  const int rows = count, units = (int)(p.rows.row_bytes / sizeof(U));
  int still = 0;  // nodes that stay where they are
  while (still < rows && path[still] == still) ++still;
  // unit i: row i % moved of the moved ones, column i / moved
  const int moved = rows - still, columns = moved > 0 ? max(kAcceptThreads * kAcceptPieces / moved, 1) : 1;
  for (int c0 = 0; moved > 0 && c0 < units; c0 += columns) {
    const int wide = min(columns, units - c0), all = wide * moved;
    U v[kAcceptPieces];
#pragma unroll
    for (int k = 0; k < kAcceptPieces; ++k) {
      const int i = threadIdx.x + k * kAcceptThreads, r = still + i / wide;
      if (i < all) v[k] = reinterpret_cast<const U*>(moved_row(p.rows, s, begin, L - n + path[r]))[c0 + i % wide];
    }
    rows_read();
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kAcceptPieces; ++k) {
      const int i = threadIdx.x + k * kAcceptThreads, r = still + i / wide;
      if (i < all) reinterpret_cast<U*>(moved_row(p.rows, s, begin, L - n + r))[c0 + i % wide] = v[k];
    }
  }
  if (threadIdx.x == 0) p.rows.lens[s] = L - n + rows;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

}  // namespace

hipError_t launch_tree_queries(const TreeQueries& p, hipStream_t stream) {
  const int elems = p.nh * (p.dn > p.dR / 2 ? p.dn : p.dR / 2);
  const unsigned shares = p.q_nope || p.q_rope ? (unsigned)((elems + kElems - 1) / kElems) : 1;
  if (shares > kMostBlocksYZ) return hipErrorInvalidValue;
  const auto k = p.vec && p.dn % 4 == 0 && p.dR % 8 == 0 ? tree_queries_kernel<4> : tree_queries_kernel<1>;
  return in_grids(p.q.tokens, most_blocks(256), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL(k, dim3(blocks, shares), dim3(256), 0, stream, p, first);
  });
}

hipError_t launch_plain_tree(const PlainTree& p, hipStream_t stream) {
  const int64_t items = (int64_t)p.src.num_seqs * p.nodes * p.nh;
  if (items > INT32_MAX || !generic_prompt_supported(p.dc, p.dR)) return hipErrorInvalidValue;
  return in_grids(items, most_blocks(256), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL(plain_tree_kernel, dim3(blocks), dim3(256), 0, stream, p, first);
  });
}

hipError_t launch_accept(const AcceptProblem& p, hipStream_t stream) {
  const int unit = moved_unit(p.rows);
  const auto k = unit == 16  ? accept_kernel<u32x4>
                 : unit == 8 ? accept_kernel<uint64_t>
                 : unit == 4 ? accept_kernel<uint32_t>
                 : unit == 2 ? accept_kernel<uint16_t>
                             : accept_kernel<uint8_t>;
  return in_grids(p.rows.num_seqs, most_blocks(kAcceptThreads), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL(k, dim3(blocks), dim3(kAcceptThreads), 0, stream, p, first);
  });
}

}  // namespace la
