// The attention weight that cache rows get (la_weigh_kv):
//   w[s, p] += sum_{t, h} 2^(x[t, h, p] - m[t, h]) / l[t, h],  x = scale log2(e) (q_abs . c_t[p] + q_rope . RoPE(k_rope[p], p)),
// over the sequence's last tokens t (causal) and all heads h, m the maximum of a
// row of x and l the sum of its 2^(x - m). The weights are sums over many steps that rank rows
// against each other, so they and the scores are kept to fp32. (m and l stay apart: m + log2 l has only
// what m's size leaves of l, nothing where m passes 2^24.)
#include "la_draft.hpp"

#include <type_traits>

namespace la {
namespace {

constexpr float kNoScore = -3.402823466e38f;  // no finite score is below
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
  return scaled_score(wave_sum(d), p.scale_log2);
}
__device__ inline void plain_query(const WeighProblem& p, int64_t item, int lane, float (&q)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) q[i] = lane + 64 * i < p.dc ? p.q_abs[item * p.dc + lane + 64 * i] : 0.f;
}

// The plain form, for any type and head shape: a workgroup of 4 waves per
// (token, head) for maxima and sums, then a wave per row that goes through
// all (token, head) again. Sums in a fixed order. Bound by the rows' and the
// queries' way from the L2.
__global__ __launch_bounds__(256) void plain_sums_kernel(WeighProblem p, int64_t first) {
  __shared__ float ml[4][2];
  const uint32_t item = (uint32_t)first + blockIdx.x;
  const int token = (int)(item / p.nh), s = token / p.tokens, j = token % p.tokens;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int keys = source_rows(p.src, s) - p.tokens + j + 1;
  float q[16], m = kNoScore, l = 0.f;
  plain_query(p, item, lane, q);
  for (int64_t k = wave; k < keys; k += 4) {  // (up to 2^31 - 1 rows)
    const float x = plain_score(p, q, p.q_rope + item * (int64_t)p.dR, s, (int)k, lane), up = fmaxf(m, x);
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
    p.sums[2 * (int64_t)item] = keys > 0 ? top : INFINITY;  // no row gets anything of a token that sees none
    p.sums[2 * (int64_t)item + 1] = keys > 0 ? 1.f / total : 0.f;
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
    sum += exp2f(plain_score(p, q, p.q_rope + item * p.dR, s, (int)k, lane) - p.sums[2 * item]) * p.sums[2 * item + 1];
  }
  const int64_t at = (p.src.offsets ? source_begin(p.src, s) : (int64_t)s * p.src.region) + k;
  if (lane == 0) p.weights[at] += sum;
}

// ---- the matrix form ----------------------------------------------------------------------------------

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lchar;

// Two parts of a value in the products' type: hi + lo. fp16 has more bits than bf16 and a
// narrow range, so there
// - queries come times kUp, and the pieces of a row (32 latent columns, the rope part) that are
//   too large or too small then are divided by powers of two (fit_f16). When the products' operands of
//   such a row are loaded they are brought to one divisor, which leaves the row's largest element near
//   fp16's and is taken off the scores: any queries that fp32 holds will do (elements below 2^-22 of a
//   row's largest lose bits of 2^-18 of them);
// - rotated keys come in halves (they reach sqrt(2) times the largest fp16 number) and what is
//   left of them times kLow, against queries divided by it: it would be subnormal, or nothing, in
//   small keys.
template <typename T>
struct Mm;
template <>
struct Mm<__hip_bfloat16> {
  typedef bf16x8 vec;
  typedef __bf16 elem;
  static constexpr float kUp = 1.f, kKey = 1.f, kLow = 1.f;
  static __device__ inline f32x16 mma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mm<__half> {
  typedef f16x8 vec;
  typedef _Float16 elem;
  static constexpr float kUp = 64.f, kKey = 1.f / kUpRope, kLow = 2048.f;
  static __device__ inline f32x16 mma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <typename T>
__device__ inline void split(float x, typename Mm<T>::elem& hi, typename Mm<T>::elem& lo, float low = 1.f) {
  hi = (typename Mm<T>::elem)x;
  lo = (typename Mm<T>::elem)((x - (float)hi) * low);
}

// Tiles of 32 rows of the piece's sequences, counted over them, shared out evenly:
// span w of W has [w T / W, (w + 1) T / W), one tile at least (W <= T). The lengths are on the device, so
// every wave sums them itself. Tiles past p.tiles (of packed sequences whose offsets are not in order) are left out:
// every index below is below that then.
struct Spans {
  const WeighProblem& p;
  __device__ int tiles(int i) const {  // of the piece's sequence i
    return i < p.seqs ? (source_rows(p.src, p.seq0 + i) + kWeighKeys - 1) / kWeighKeys : 0;
  }
  __device__ int total() const {
    int t = 0;
    for (int i = wave_lane(); i < p.seqs; i += 64) t = min(t + tiles(i), p.tiles);
    return (int)min((uint32_t)wave_sum_i(t), (uint32_t)p.tiles);  // (64 numbers below 2^26)
  }
  // Sequence of tile t (< total), its first tile and tiles; false only if the lengths change meanwhile. (The sums up to
  // the first that passes t stay below 2^27.)
  __device__ bool find(int t, int* seq, int* first, int* n) const {
    int before = 0;
    for (int i0 = 0; i0 < p.seqs; i0 += 64) {
      const int mine = tiles(i0 + wave_lane()), end = wave_scan(mine);
      const uint64_t past = __builtin_amdgcn_ballot_w64(before + end > t);
      if (past) {
        const int k = __builtin_ctzll(past);
        *seq = i0 + k;
        *n = __builtin_amdgcn_readlane(mine, k);
        *first = before + __builtin_amdgcn_readlane(end, k) - *n;
        return true;
      }
      before += __builtin_amdgcn_readlane(end, 63);
    }
    return false;
  }
  // The next one with tiles.
  __device__ bool next(int* seq, int* first, int* n) const {
    *first += *n;
    do {
      if (++*seq >= p.seqs) return false;
      *n = tiles(*seq);
    } while (*n == 0);
    return true;
  }
  static __device__ int begin(int w, int T, int W) { return (int)((int64_t)w * T / W); }
  static __device__ int of(int t, int T, int W) { return (int)((((int64_t)t + 1) * W - 1) / T); }  // the span that has tile t
};

// One tile in LDS: 32 rows of 1024 B whose starts are spread over the banks (every
// read takes one 16-B piece of each row), and the rotated rope keys in two parts,
// 128-B rows with their 16-B pieces permuted.
constexpr int kPitch = 1088;
__host__ __device__ constexpr int row_at(int r) { return r * kPitch + 16 * ((r >> 2) & 3); }
__device__ inline int rope_piece(int row, int piece) { return row * 128 + 16 * (piece ^ ((row >> 1) & 7)); }
constexpr int kRopeHi = (row_at(31) + 1024 + 127) / 128 * 128, kRopeLo = kRopeHi + 32 * 128, kTile = kRopeLo + 32 * 128;

// What a wave of kW holds of a tile on its way to LDS: the latent parts of its kS = 32 / kW rows,
// 16 (8-bit rows: 8) B of each per lane, and kP pairs of the rope part of row lane / kLR.
template <bool kFp8, int kW>
struct Staged {
  static constexpr int kS = 32 / kW, kLR = 64 / kS, kP = 32 / kLR;
  typedef typename std::conditional<kFp8, u32x2, u32x4>::type cvec;
  typedef typename std::conditional<(kFp8 ? kP : 2 * kP) == 8, u32x2,
                                    typename std::conditional<(kFp8 ? kP : 2 * kP) == 4, uint32_t, uint16_t>::type>::type kvec;
  typedef float pvec __attribute__((ext_vector_type(kP)));
  cvec c[kS];
  kvec ka, kb;
  pvec cs, sn;
};
// A sequence's rows: the first (contiguous caches) and the last, and its block table.
struct Rows {
  int64_t begin;
  const int32_t* table;
  int last;
};
// Position of the lane's part of tile t (past the last row: that one), and its block
// table's entry: looked up a tile before its loads, so that it has arrived by then.
template <int kW>
__device__ inline int stage_pos(const Rows& r, int t, int wave, int lane) {
  return min(kWeighKeys * t + 32 / kW * wave + lane / (2 * kW), r.last);
}
template <int kW>
__device__ inline int stage_entry(const WeighProblem& p, const Rows& r, int t, int wave, int lane) {
  return r.table ? r.table[stage_pos<kW>(r, t, wave, lane) / p.src.block_size] : 0;
}
template <bool kFp8, int kW>
__device__ inline void stage_load(const WeighProblem& p, const Rows& r, Staged<kFp8, kW>& x, int entry, int t, int wave, int lane) {
  typedef Staged<kFp8, kW> S;
  constexpr int kRowB = kFp8 ? 576 : 1152;
  const int pos = stage_pos<kW>(r, t, wave, lane);
  int64_t src = r.begin + pos;
  if (r.table) src = clamp64(entry, 0, p.src.pool_blocks - 1) * p.src.block_size + pos % p.src.block_size;
  const int64_t at = src * kRowB;
  const char* const kv = static_cast<const char*>(p.src.kv);
#pragma unroll
  for (int i = 0; i < S::kS; ++i) {
    const int64_t row = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(at >> 32), S::kLR * i) << 32 |
                        (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)at, S::kLR * i);
    x.c[i] = reinterpret_cast<const typename S::cvec*>(kv + row)[lane];
  }
  int part = lane;
  asm volatile("" : "+v"(part));  // (the address with it, held through the tiles' loop, was spilled)
  const char* const rope = kv + at + (kFp8 ? 512 : 1024) + sizeof(typename S::kvec) * (part % S::kLR);
  x.ka = *reinterpret_cast<const typename S::kvec*>(rope);
  x.kb = *reinterpret_cast<const typename S::kvec*>(rope + (kFp8 ? 32 : 64));
  const int64_t rp = source_rope_row(p.src, pos) * 32 + S::kP * (lane % S::kLR);
  x.cs = *reinterpret_cast<const typename S::pvec*>(p.src.cos + rp);
  x.sn = *reinterpret_cast<const typename S::pvec*>(p.src.sin + rp);
}
template <typename T, bool kFp8, int kW>
__device__ inline void stage_store(const Staged<kFp8, kW>& x, lchar* L, int wave, int lane) {
  typedef Staged<kFp8, kW> S;
  typedef typename Mm<T>::elem elem;
  auto put = [&](int at, auto v) { *reinterpret_cast<__attribute__((address_space(3))) decltype(v)*>(L + at) = v; };
  const int row0 = row_at(S::kS * wave) + 16 * lane;  // row i of the wave is 1088 i + 16 (i / 4) on
#pragma unroll
  for (int i = 0; i < S::kS; ++i) {
    u32x4 y;
    if constexpr (kFp8) {
      y[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.c[i][0], 1.f, false));
      y[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.c[i][0], 1.f, true));
      y[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.c[i][1], 1.f, false));
      y[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.c[i][1], 1.f, true));
    } else {
      y = x.c[i];
    }
    put(row0 + kPitch * i + 16 * (i >> 2), y);
  }
  // element e of a lane's share
  auto word = [](const typename S::kvec& v, int i) -> uint32_t {
    if constexpr (sizeof(v) == 8) return v[i];
    else return (uint32_t)v;
  };
  auto value = [&](const typename S::kvec& v, int e) -> float {
    if constexpr (kFp8) {
      const uint32_t w = word(v, 0);
      const auto two = (e & 2) ? __builtin_amdgcn_cvt_pk_f32_fp8(w, true) : __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
      return two[e & 1];
    } else {
      return (float)__builtin_bit_cast(elem, (uint16_t)(word(v, e >> 1) >> (16 * (e & 1))));
    }
  };
  typedef elem evec __attribute__((ext_vector_type(S::kP)));
  evec ah, al, bh, bl;
#pragma unroll
  for (int e = 0; e < S::kP; ++e) {
    const float a = value(x.ka, e), b = value(x.kb, e);
    elem h, l;
    split<T>((a * x.cs[e] - b * x.sn[e]) * Mm<T>::kKey, h, l, Mm<T>::kLow);
    ah[e] = h, al[e] = l;
    split<T>((a * x.sn[e] + b * x.cs[e]) * Mm<T>::kKey, h, l, Mm<T>::kLow);
    bh[e] = h, bl[e] = l;
  }
  const int row = S::kS * wave + lane / S::kLR, i0 = S::kP * (lane % S::kLR);
  const int pa = rope_piece(row, i0 >> 3) + 2 * (i0 & 7), pb = rope_piece(row, 4 + (i0 >> 3)) + 2 * (i0 & 7);
  put(kRopeHi + pa, ah);
  put(kRopeLo + pa, al);
  put(kRopeHi + pb, bh);
  put(kRopeLo + pb, bl);
}

// Scores of a span's tiles against 128 (32 kWR) rows of queries, and their partial
// maxima and sums of exponentials.
//
// Precision: a score has to hold fp32's worth, since weights are compared with each
// other; fp32 matrix instructions have a sixteenth of the 16-bit ones' rate.
// Cache rows are 16-bit numbers (8-bit ones widen exactly to fp16), so the queries go in as
// two 16-bit parts, hi and what is left, whose products with a row are exact and
// summed in fp32: 2 products for the latent part, 3 for the rope part, whose
// rotated keys have two parts as well. bf16 leaves 2^-18 of an operand, fp16 less.
//
// kWR of the kW waves have 32 rows of queries each, with their operands in registers
// for the whole segment; the kKD = kW / kWR others of a row block take shares of the
// contraction, summed through LDS. So all matrix cores work whatever the rows, and
// a SIMD has two waves (256 registers each), one's other work under the other's
// products: up to 64 rows in two workgroups of 4 waves per CU, more in one of 8, whose
// tiles serve 128 rows (32 x 8192 rows, 128 heads: a call 154 us when they were compared; in the form of 64 rows,
// which loads and stages every tile twice, 171). Tiles go HBM -> registers -> LDS, the
// next one on its way during the products; a buffer of its own for it and for the sums
// leaves one barrier a tile (with two 158).
// What bounds it: at 128 rows the round of staging, products, sums and exponentials of a
// tile, 114 us for those 302 MB and 82 GFLOP (hi and lo): 2.7 TB/s and 0.72 PFLOP/s, each
// half of its rate (fp16 rows, with their queries' and keys' scaling, 145 a call for 141, 8-bit ones 134 for 128 as
// bf16). With 16 rows (64 x 300 to 4000 8-bit rows) 27 us, 2.7 TB/s of rows, the
// same round with a quarter of the products; 1001 rows of one sequence 11 us, a few round trips.
constexpr int weigh_sums(int kWR, int kW) { return (kW / kWR == 2 ? 2048 : 4096) * kW; }
template <typename T, bool kFp8, int kWR, int kW>
__global__ __launch_bounds__(64 * kW, 2) void weigh_scores_kernel(WeighProblem p, int row_blocks) {
  typedef typename Mm<T>::vec vec;
  typedef typename Mm<T>::elem elem;
  typedef __attribute__((address_space(3))) f32x4 lvec;
  constexpr int kKD = kW / kWR;           // shares of the contraction
  constexpr int kC = 32 / kKD;            // latent steps of 16 of a share
  constexpr int kR = 4 / kKD;             // rope steps
  constexpr int kN = 16 / kKD;            // scores of a lane after the sum
  constexpr bool kTwo = kW == 8;          // two buffers of a tile and of its sums: one barrier a tile
  constexpr int kSums = weigh_sums(kWR, kW);
  constexpr bool kFit = Mm<T>::kUp != 1.f;
  static_assert(kKD == 2 || kKD == 4, "the waves meet at the sums, behind a tile's last read");
  extern __shared__ __attribute__((aligned(1024))) char weigh_lds[];
  lchar* const L = (lchar*)weigh_lds;
  lchar* const sums0 = L + (kTwo ? 2 : 1) * kTile;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  // what a row's products are multiplied by (in LDS, a word per row and wave: a register more is spilled)
  typedef __attribute__((address_space(3))) float lfloat;
  lfloat* const back = reinterpret_cast<lfloat*>(sums0 + (kTwo ? 2 : 1) * kSums) + 32 * wave + (lane & 31);
  const int wr = wave % kWR, kd = wave / kWR, r32 = lane & 31, g = lane >> 5;
  // an eighth of the items to each XCD, row groups of a span together
  const int groups = (row_blocks + kWR - 1) / kWR, items = p.spans * groups, per = (items + 7) / 8;
  const int item = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || item >= items) return;
  const int span = item / groups, block = item % groups * kWR + wr;
  const int row = 32 * block + r32;
  const bool valid = row < p.count;
  const Spans sp{p};
  const int T_all = sp.total(), W = min(p.spans, T_all);
  if (span >= W) return;
  int t = Spans::begin(span, T_all, W);
  const int t_end = Spans::begin(span + 1, T_all, W);
  int i, first, n;
  if (!sp.find(t, &i, &first, &n)) return;
  while (true) {
    const int s = p.seq0 + i, len = source_rows(p.src, s), end = min(t_end, first + n);
    Staged<kFp8, kW> x;  // the next tile, and the table's entry of the one after it
    auto tile = [&](int u) { return min(u, end - 1) - first; };
    const Rows from{p.src.block_table ? 0 : source_begin(p.src, s),
                    p.src.block_table ? p.src.block_table + (int64_t)s * p.src.blocks_per_seq : nullptr, len - 1};
    stage_load(p, from, x, stage_entry<kW>(p, from, tile(t), wave, lane), tile(t), wave, lane);
    int entry = stage_entry<kW>(p, from, tile(t + 1), wave, lane);
    // ---- the queries' operands: [16 k + 8 g .. + 7] of the row, 1 KB per step ----
    vec qh[kC + kR], ql[kC + kR];
    {
      const int64_t at = (((int64_t)s * qprep_rows_per_seq(p.tokens * p.nh) + p.row0) / 32 + min(block, row_blocks - 1)) * (32 * kQPrepRow);
      const elem *const q = static_cast<const elem*>(p.q_prep) + at + 8 * lane, *const low = q + p.low;
#pragma unroll
      for (int k = 0; k < kC + kR; ++k) {
        const int step = 512 * (k < kC ? kC * kd + k : 32 + kR * kd + k - kC);
        qh[k] = *reinterpret_cast<const vec*>(q + step);
        ql[k] = *reinterpret_cast<const vec*>(low + step);
      }
    }
    if constexpr (kFit) {
      typedef uint32_t words __attribute__((ext_vector_type(4), aligned(4)));
      const uint8_t* const pieces = p.most + ((int64_t)s * qprep_rows_per_seq(p.tokens * p.nh) + p.row0 + min(row, p.count - 1)) * kMostRow;
      const words first = *reinterpret_cast<const words*>(pieces);
      const uint32_t last = pieces[16];
      auto piece = [&](int k) { return k < 16 ? (int)(first[k >> 2] >> (8 * (k & 3)) & 255) : (int)last; };
      int most = 0;
      bool fits = true;
#pragma unroll
      for (int k = 0; k < kMostPieces; ++k) {
        most = max(most, piece(k));
        fits = fits && fit_f16(piece(k)) == 0;
      }
      const int by = fits ? 0 : top_f16(most);
      *back = power_of_2(by) * (1.f / Mm<T>::kUp);  // (the same from both halves' lanes)
      if (__builtin_amdgcn_ballot_w64(!fits) != 0) {
        const uint32_t* const own = reinterpret_cast<const uint32_t*>(pieces + kC / 2 * kd);
#pragma unroll
        for (int k = 0; k < kC + kR; ++k) {
          const int e = fit_f16(k < kC ? (int)(own[k / 8] >> (8 * (k / 2 & 3)) & 255) : (int)last) - by;
          const int e1 = min(max(e, -14), 14);  // in two steps, each a power of two that fp16 holds (or what is left is nothing)
          const elem f1 = (elem)power_of_2(e1), f2 = (elem)power_of_2(max(e - e1, -100));
          qh[k] = qh[k] * f1 * f2;
          ql[k] = ql[k] * f1 * f2;
        }
      }
    }
    int own_score = 32 * r32 + 2 * kN * kd + 4 * g;  // of a tile's
    asm volatile("" : "+v"(own_score));  // (the address with it, made before the operands, was spilled)
    // keys that the row's token sees
    const int sees = len - p.tokens + (int)((uint32_t)(p.row0 + row) / (uint32_t)p.nh) + 1;
    float m = kNoScore, l = 0.f;
    if constexpr (kTwo) {
      stage_store<T>(x, L, wave, lane);
      stage_load(p, from, x, entry, tile(t + 1), wave, lane);
      entry = stage_entry<kW>(p, from, tile(t + 2), wave, lane);
      lds_barrier();
    }
    for (int u = t; u < end; ++u) {
      // (the waves have met behind the last read of the tile before, at its sums)
      stage_store<T>(x, L + (kTwo ? (u + 1 - t) & 1 : 0) * kTile, wave, lane);
      stage_load(p, from, x, entry, tile(u + (kTwo ? 2 : 1)), wave, lane);
      entry = stage_entry<kW>(p, from, tile(u + (kTwo ? 3 : 2)), wave, lane);
      if constexpr (!kTwo) lds_barrier();
      const lchar* const b = L + (kTwo ? (u - t) & 1 : 0) * kTile;
      lchar* const sums = sums0 + (kTwo ? (u - t) & 1 : 0) * kSums;
      f32x16 acc = {};
      uint32_t below = __builtin_bit_cast(uint16_t, (elem)(1.f / Mm<T>::kLow));
      asm volatile("" : "+s"(below));  // (the products with it, made before the loop, were spilled)
      auto operand = [&](int k) -> vec {  // keys r32, elements [16 k + 8 g .. + 7]
        const int at = k < kC ? row_at(r32) + 32 * (kC * kd + k) + 16 * g
                       : k < kC + kR ? kRopeHi + rope_piece(r32, 2 * (kR * kd + k - kC) + g)
                                     : kRopeLo + rope_piece(r32, 2 * (kR * kd + k - kC - kR) + g);
        return *reinterpret_cast<const __attribute__((address_space(3))) vec*>(b + at);
      };
      constexpr int kSteps = kC + 2 * kR, kAhead = 3;
      vec a[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) a[k] = operand(k);
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const vec v = a[k % kAhead];
        if (k < kC + kR) acc = Mm<T>::mma(v, ql[k], acc);
        if (k < kC + kR) acc = Mm<T>::mma(v, qh[k], acc);
        else acc = Mm<T>::mma(v, kFit ? qh[k - kR] * __builtin_bit_cast(elem, (uint16_t)below) : qh[k - kR], acc);
        if (k + kAhead < kSteps) a[k % kAhead] = operand(k + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
      settle(acc);
      // lane: row r32, keys 8 (e / 4) + 4 g + e % 4; this share's are quads kN / 4 kd and on
      float sc[kN];
      const float to_score = kFit ? *back : 1.f;
      auto quad = [&](int q) {
        return f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
      };
      if constexpr (kKD == 2) {  // the other's quads to it, its for this wave back
        lchar* const mine = sums + 2048 * wave + 16 * lane;
#pragma unroll
        for (int q = 0; q < 2; ++q) *reinterpret_cast<lvec*>(mine + 1024 * q) = kd == 0 ? quad(2 + q) : quad(q);
        lds_barrier();
        const lchar* const its = sums + 2048 * (wr + kWR * (1 - kd)) + 16 * lane;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const f32x4 v = *reinterpret_cast<const lvec*>(its + 1024 * q), own = kd == 0 ? quad(q) : quad(2 + q);
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[4 * q + e] = (own[e] + v[e]) * to_score;
        }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) *reinterpret_cast<lvec*>(sums + 4096 * wave + 1024 * q + 16 * lane) = quad(q);
        lds_barrier();
#pragma unroll
        for (int q = 0; q < kN / 4; ++q) {
          f32x4 v = {};
#pragma unroll
          for (int w = 0; w < kKD; ++w)
            v += *reinterpret_cast<const lvec*>(sums + 4096 * (wr + kWR * w) + 1024 * (kN / 4 * kd + q) + 16 * lane);
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[4 * q + e] = v[e] * to_score;
        }
      }
      const int key0 = kWeighKeys * (u - first) + 2 * kN * kd + 4 * g;
      const int most = min(len, sees) - key0;
      if (kWeighKeys * (u - first + 1) > len - p.tokens + p.row0 / p.nh + 1) {
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (8 * (e >> 2) + (e & 3) >= most) sc[e] = -INFINITY;
      }
      float top = sc[0];
#pragma unroll
      for (int e = 1; e < kN; ++e) top = fmaxf(top, sc[e]);
      const float up = fmaxf(m, top);
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < kN; ++e) sum += __builtin_amdgcn_exp2f(sc[e] - up);
      l = l * __builtin_amdgcn_exp2f(m - up) + sum;
      m = up;
      if (valid) {
        float* const to = p.scores + ((int64_t)u * row_blocks + block) * 1024 + own_score;
#pragma unroll
        for (int q = 0; q < kN / 4; ++q)
          *reinterpret_cast<f32x4*>(to + 8 * q) = f32x4{sc[4 * q], sc[4 * q + 1], sc[4 * q + 2], sc[4 * q + 3]};
      }
    }
    lds_barrier();  // every wave is done with the segment
    // ---- the segment's share of the rows' sums ----
    {
      auto join = [&](float m2, float l2) {
        const float up = fmaxf(m, m2);
        l = l * __builtin_amdgcn_exp2f(m - up) + l2 * __builtin_amdgcn_exp2f(m2 - up);
        m = up;
      };
      const auto sm = __builtin_amdgcn_permlane32_swap(u_of(m), u_of(m), false, false);
      const auto sl = __builtin_amdgcn_permlane32_swap(u_of(l), u_of(l), false, false);
      m = f_of(sm[0]), l = f_of(sl[0]);
      join(f_of(sm[1]), f_of(sl[1]));
      lfloat* const ml = reinterpret_cast<lfloat*>(sums0) + 64 * wave;
      if (g == 0) ml[r32] = m, ml[32 + r32] = l;
      lds_barrier();
#pragma unroll
      for (int w = 1; w < kKD; ++w) {
        const lfloat* const o = reinterpret_cast<const lfloat*>(sums0) + 64 * (wr + kWR * w);
        if (kd == 0) join(o[r32], o[32 + r32]);
      }
      if (kd == 0 && g == 0 && block < row_blocks) {
        int r = r32;
        asm volatile("" : "+v"(r));  // (the address, made before the loop, was spilled)
        float* const to = p.part + (int64_t)(span + i) * 2 * 32 * row_blocks + 32 * block + r;
        to[0] = m;
        to[32 * row_blocks] = l;
      }
    }
    t = end;
    if (t >= t_end || !sp.next(&i, &first, &n)) return;
  }
}

// The second kernel: rows' maxima and sums from their parts, then a wave per
// tile adds the exponentials of its scores over the rows, in their order. Bound by
// the scores' way back (32 x 8192 rows, 128 heads: 134 MB in 30 us, 4.5 TB/s).
__global__ __launch_bounds__(256) void weigh_sum_kernel(WeighProblem p, int row_blocks) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  extern __shared__ __attribute__((aligned(8))) char weigh_sums_lds[];
  f32x2* const all = reinterpret_cast<f32x2*>(weigh_sums_lds);  // of every row its maximum, and 1 / its sum
  __shared__ f32x4 part[4][8];
  __shared__ int bad[2];  // whether a row's sum is not a number (of a segment, and the next)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Spans sp{p};
  const int T_all = sp.total(), W = min((int)gridDim.x, T_all), W1 = min(p.spans, T_all), w = blockIdx.x;
  if (w >= W) return;
  int t = Spans::begin(w, T_all, W);
  const int t_end = Spans::begin(w + 1, T_all, W);
  int i, first, n;
  if (!sp.find(t, &i, &first, &n)) return;
  const int rows = p.count;
  if (threadIdx.x == 0) bad[0] = 0;
  for (int turn = 0;; turn ^= 1) {
    const int s = p.seq0 + i, len = source_rows(p.src, s), end = min(t_end, first + n);
    const int c0 = Spans::of(first, T_all, W1), c1 = Spans::of(min(first + n, T_all) - 1, T_all, W1);
    __syncthreads();
    if (threadIdx.x == 0) bad[turn ^ 1] = 0;
    for (int r = threadIdx.x; r < 32 * row_blocks; r += 256) {
      float m = kNoScore, l = 0.f;
      constexpr int kOnce = 8;  // partial sums whose loads go out together
      if (r < rows)
        for (int c = c0; c <= c1; c += kOnce) {
          float m2[kOnce], l2[kOnce], up = m;
#pragma unroll
          for (int k = 0; k < kOnce; ++k) {
            const float* const from = p.part + (int64_t)(min(c + k, c1) + i) * 2 * 32 * row_blocks + r;
            m2[k] = from[0];
            l2[k] = c + k <= c1 ? from[32 * row_blocks] : 0.f;
          }
#pragma unroll
          for (int k = 0; k < kOnce; ++k) up = fmaxf(up, m2[k]);
          l *= exp2f(m - up);
#pragma unroll
          for (int k = 0; k < kOnce; ++k) l += l2[k] * exp2f(m2[k] - up);
          m = up;
        }
      // rows past the last, and tokens that see nothing, give nothing
      all[r] = l == 0.f ? f32x2{INFINITY, 0.f} : f32x2{m, 1.f / l};
      if (l != l) bad[turn] = 1;
    }
    __syncthreads();
    const bool strict = bad[turn];
    // a tile per wave, or (many rows) a quarter of a tile's row blocks
    const bool shared = row_blocks >= 8;
    const int b0 = shared ? wave : 0, db = shared ? 4 : 1;
    for (int u = shared ? t : t + wave; u < end; u += shared ? 1 : 4) {
      const float* const from = p.scores + (int64_t)u * row_blocks * 1024 + 4 * lane;
      f32x4 sum = {};
      // hidden rows' scores are -infinity: they get nothing also from a token whose sum is not a number
      auto add = [&](auto strict) {
#pragma unroll 4
        for (int b = b0; b < row_blocks; b += db) {
          f32x4 v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = *reinterpret_cast<const f32x4*>(from + 1024 * b + 256 * q);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int r = 32 * b + 8 * q + (lane >> 3);
            const f32x2 e = all[r];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              sum[k] += r < rows && (!strict.value || v[q][k] != -INFINITY) ? __builtin_amdgcn_exp2f(v[q][k] - e[0]) * e[1] : 0.f;
          }
        }
      };
      if (strict) add(std::true_type());
      else add(std::false_type());
#pragma unroll
      for (int o = 8; o < 64; o <<= 1)
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += __shfl_xor(sum[k], o, 64);
      if (shared) {
        __syncthreads();  // (the sums of the tile before are read)
        if (lane < 8) part[wave][lane] = sum;
        __syncthreads();
        if (wave > 0) continue;
        if (lane < 8) sum = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
      }
      const int key = kWeighKeys * (u - first) + 4 * lane;
      if (lane < 8) {
        float* const to = p.weights + (p.src.offsets ? source_begin(p.src, s) : (int64_t)s * p.src.region);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (key + k < len) to[key + k] += sum[k];
      }
    }
    t = end;
    if (t >= t_end || !sp.next(&i, &first, &n)) return;
  }
}

template <typename T, bool kFp8, int kWR, int kW>
hipError_t scores_t(const WeighProblem& p, int row_blocks, hipStream_t stream) {
  constexpr int lds = (kW == 8 ? 2 : 1) * (kTile + weigh_sums(kWR, kW)) + (Mm<T>::kUp != 1.f ? 128 * kW : 0);
  static OncePerDevice once;
  const auto k = weigh_scores_kernel<T, kFp8, kWR, kW>;
  const hipError_t e = allow_lds(once, reinterpret_cast<const void*>(k), lds);
  if (e != hipSuccess) return e;
  const int64_t items = (int64_t)p.spans * ((row_blocks + kWR - 1) / kWR);
  hipLaunchKernelGGL(k, dim3((unsigned)(8 * ((items + 7) / 8))), dim3(64 * kW), lds, stream, p, row_blocks);
  return hipGetLastError();
}
template <typename T, bool kFp8>
hipError_t scores_w(const WeighProblem& p, int row_blocks, hipStream_t stream) {
  if (row_blocks == 1) return scores_t<T, kFp8, 1, 4>(p, row_blocks, stream);
  if (row_blocks == 2) return scores_t<T, kFp8, 2, 4>(p, row_blocks, stream);
  return scores_t<T, kFp8, 4, 8>(p, row_blocks, stream);
}

// Queries' operands from absorbed fp32 ones, where the absorption does not write them: 8 elements of a row per thread, the
// 4 of a piece (8 of the rope part) next to one another in a wave.
template <typename T>
__global__ __launch_bounds__(256) void weigh_queries_kernel(WeighProblem p, int64_t first) {
  typedef typename Mm<T>::elem elem;
  const int64_t n = (int64_t)p.src.num_seqs * p.tokens * p.nh * (kQPrepRow / 8), i = (first + blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;  // (whole rows)
  const int64_t row = i / (kQPrepRow / 8);
  const int j = 8 * (int)(i % (kQPrepRow / 8)), each = p.tokens * p.nh;
  const float* const from = j < 512 ? p.q_abs + row * 512 + j : p.q_rope + row * 64 + j - 512;
  const int64_t at = qprep_index(row / each * qprep_rows_per_seq(each) + row % each, j);
  elem* const to = static_cast<elem*>(const_cast<void*>(p.q_prep)) + at;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = from[e] * (p.scale_log2 * Mm<T>::kUp) * (j < 512 ? 1.f : 1.f / Mm<T>::kKey);
  if constexpr (Mm<T>::kUp != 1.f) {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
    m = fmaxf(m, __shfl_xor(m, 1, 64));
    m = fmaxf(m, __shfl_xor(m, 2, 64));
    const float wide = __shfl_xor(m, 4, 64);
    if (j >= 512) m = fmaxf(m, wide);
    if (j < 512 ? j % 32 == 0 : j == 512)
      p.most[(row / each * qprep_rows_per_seq(each) + row % each) * kMostRow + j / 32] = (uint8_t)exponent_of(m);
    const float fit = power_of_2(-fit_f16(exponent_of(m)));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= fit;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    elem h, l;
    split<T>(v[e], h, l);
    to[e] = h;
    to[p.low + e] = l;
  }
}

}  // namespace

float weigh_query_scale(const WeighProblem& p) {
  return p.scale_log2 * (weigh_f16(p.src.kv_dtype) ? Mm<__half>::kUp : Mm<__hip_bfloat16>::kUp);
}

hipError_t launch_weigh_queries(const WeighProblem& p, hipStream_t stream) {
  const int64_t n = (int64_t)p.src.num_seqs * p.tokens * p.nh * (kQPrepRow / 8);
  const auto k = weigh_f16(p.src.kv_dtype) ? weigh_queries_kernel<__half> : weigh_queries_kernel<__hip_bfloat16>;
  return in_grids((n + 255) / 256, most_blocks(256), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL(k, dim3(blocks), dim3(256), 0, stream, p, first);
  });
}

hipError_t launch_weigh_plain(const WeighProblem& p, hipStream_t stream) {
  const int64_t items = (int64_t)p.src.num_seqs * p.tokens * p.nh;
  if (items > INT32_MAX || p.dc > kLatent) return hipErrorInvalidValue;
  hipError_t e = in_grids(items, most_blocks(256), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL(plain_sums_kernel, dim3(blocks), dim3(256), 0, stream, p, first);
  });
  const int64_t most = p.src.offsets ? p.src.total_rows : p.src.region;
  for (int s = 0; s < p.src.num_seqs && e == hipSuccess; ++s)
    e = in_grids((most + 3) / 4, most_blocks(256), [&](int64_t first, unsigned blocks) {
      hipLaunchKernelGGL(plain_weigh_kernel, dim3(blocks), dim3(256), 0, stream, p, s, first);
    });
  return e;
}

bool weigh_mfma_supported(const WeighProblem& p) {
  if (p.src.kv_dtype == LA_DTYPE_F32 || p.dc != 512 || p.dR != 64) return false;
  // 16-byte loads of rows and tables
  if (((reinterpret_cast<uintptr_t>(p.src.kv) | reinterpret_cast<uintptr_t>(p.src.cos) | reinterpret_cast<uintptr_t>(p.src.sin)) & 15) != 0)
    return false;
  return device_is_gfx950();
}

int weigh_spans(int rows, int ncu) {  // as many workgroups as run at once
  const int blocks = (rows + 31) / 32, groups = blocks <= 2 ? 1 : (blocks + 3) / 4, most = blocks <= 2 ? 2 * ncu : ncu;
  return groups < most ? most / groups : 1;
}

hipError_t launch_weigh_mfma(const WeighProblem& p, hipStream_t stream, int ncu) {
  const int row_blocks = (p.count + 31) / 32;
  hipError_t e = p.src.kv_dtype == LA_DTYPE_FP8_E4M3 ? scores_w<__half, true>(p, row_blocks, stream)
                 : p.src.kv_dtype == LA_DTYPE_BF16   ? scores_w<__hip_bfloat16, false>(p, row_blocks, stream)
                                                     : scores_w<__half, false>(p, row_blocks, stream);
  if (e != hipSuccess) return e;
  const int64_t items = row_blocks >= 8 ? p.tiles : ((int64_t)p.tiles + 3) / 4, blocks = items < 8LL * ncu ? items : 8LL * ncu;
  static_assert(8 * kWeighRows <= 64 * 1024, "LDS of a launch");
  hipLaunchKernelGGL(weigh_sum_kernel, dim3((unsigned)blocks), dim3(256), 8 * 32 * row_blocks, stream, p, row_blocks);
  return hipGetLastError();
}

}  // namespace la
