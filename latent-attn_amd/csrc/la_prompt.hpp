// Types shared by the prompt and shared-prefix kernels (la_prompt.hip,
// la_expand.hip, la_join.hip) and the C-ABI layer. Not installed.
#pragma once

#include "la_internal.hpp"

namespace la {

// Keys per tile of the expanded form. Tiles hold rows of one sequence; the
// rows past its last one are zero.
constexpr int kTileKeys = 64;
// Expanded bytes of one tile: a head's K (64 x 128) or V, and the rotated rope
// keys, which all heads share, each 16-bit, in the order that the matrix
// instructions take (below).
constexpr int kTileKBytes = kTileKeys * 128 * 2;
constexpr int kTileRBytes = kTileKeys * 64 * 2;
// Latent rows of one tile in 16 bits.
constexpr int kTileCBytes = kTileKeys * 512 * 2;

// Operand order. An instruction (v_mfma_f32_32x32x16) takes 8 elements of its
// contraction from each of two lanes per row, and any order of the contraction
// serves if both operands follow it. Accumulators come out with rows 8 b + 4 g +
// (0..3) in registers 4 b .. 4 b + 3 of lane half g, so elements e < 4 of step k
// (16 elements of the contraction) are 16 k + 4 g + e and elements e >= 4 are 16
// k + 8 + 4 g + (e - 4): then an accumulator of one product is an operand of the
// next with no lane exchange (scores -> probabilities, and expanded keys and
// values as they are stored). K of a tile: [key block of 32][step of 16 dims
// (8)][lane][8 elements], lane = key % 32 + 32 g; rope keys the same with 4
// steps; V: [dim block of 32 (4)][step of 16 keys (4)][lane][8], lane = dim % 32
// + 32 g. Every operand is one 16-B load per lane, 1 KB per wave, consecutive.
__host__ __device__ inline int operand_elem(int r, int d) {  // element (row r of 32, contraction index d of one step)
  return 8 * ((r & 31) + 32 * ((d >> 2) & 1)) + 4 * ((d >> 3) & 1) + (d & 3);
}

// Rows of sequences in a latent cache (la_prefill_args).
struct RowSource {
  const void* kv;
  int kv_dtype;
  int row_elems;  // dc + dR
  int64_t total_rows;
  int num_seqs;
  int region;              // rows of a sequence at most (offsets == nullptr)
  int stride_rows;         // rows from one region to the next (contiguous, offsets == nullptr)
  const int32_t* offsets;  // device, num_seqs + 1, or nullptr
  const int32_t* lens;     // device, num_seqs, or nullptr
  const int32_t* block_table;
  int block_size;
  int blocks_per_seq;
  int64_t pool_blocks;
  const float* cos;
  const float* sin;
  int64_t rope_rows;
  int64_t num_tiles;  // tiles of the row space below
};

__host__ __device__ inline int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// First cache row of sequence s (contiguous caches) and its rows.
__device__ inline int64_t source_begin(const RowSource& r, int s) {
  return r.offsets ? clamp64(r.offsets[s], 0, r.total_rows) : (int64_t)s * r.stride_rows;
}
__device__ inline int source_rows(const RowSource& r, int s) {
  if (s >= r.num_seqs) return 0;
  int64_t n = r.offsets ? clamp64(r.offsets[s + 1], 0, r.total_rows) - source_begin(r, s) : (int64_t)r.region;
  if (r.lens) n = n < (int64_t)r.lens[s] ? n : (int64_t)r.lens[s];
  return n < 0 ? 0 : (int)n;
}
// Tiles of the sequences: equal regions one after another; packed ones start
// at tile offset/64 + s, which leaves every sequence the tiles it needs
// (ceil(n/64) <= floor(n/64) + 1).
__device__ inline int64_t source_tile(const RowSource& r, int s) {
  if (r.offsets) return source_begin(r, s) / kTileKeys + s;
  return (int64_t)s * ((r.region + kTileKeys - 1) / kTileKeys);
}
// Sequence of a tile: the last one that starts at or before it.
__device__ inline int source_find(const RowSource& r, int64_t tile) {
  if (!r.offsets) return (int)(tile / ((r.region + kTileKeys - 1) / kTileKeys));
  int lo = 0, hi = r.num_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (source_tile(r, mid) <= tile) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// Cache row of position pos of sequence s, which has more than pos rows. Block
// ids are clamped into the pool.
__device__ inline int64_t source_row(const RowSource& r, int s, int pos) {
  if (!r.block_table) return source_begin(r, s) + pos;
  const int64_t b = clamp64(r.block_table[(int64_t)s * r.blocks_per_seq + pos / r.block_size], 0, r.pool_blocks - 1);
  return b * r.block_size + pos % r.block_size;
}
__device__ inline int64_t source_rope_row(const RowSource& r, int64_t pos) {
  return r.rope_rows > 0 && pos >= r.rope_rows ? r.rope_rows - 1 : pos;
}

// Query tokens of the sequences, packed: sequence s has [begin(s), begin(s+1)).
struct QuerySource {
  const void* q_nope;  // element (token, head, i) at token * nope_stride + head * nope_head + i
  const void* q_rope;
  int dtype;
  int64_t nope_stride, nope_head, rope_stride, rope_head;
  int rotate;             // rotate q_rope by the token's position
  int64_t tokens;
  int num_seqs;
  int per_seq;             // tokens of every sequence (offsets == nullptr)
  const int32_t* offsets;  // device, num_seqs + 1 (the first taken as 0), or nullptr
  const int32_t* prefix;   // device, num_seqs, or nullptr: rows that every token of the sequence sees
  int all;                 // every token sees every row
};
// The tokens behind the last sequence (a padded batch) are those of one more,
// which has no rows: their output rows are zero.
__device__ inline int64_t query_begin(const QuerySource& q, int s) {
  if (!q.offsets) return (int64_t)s * q.per_seq;
  return s > q.num_seqs ? q.tokens : s == 0 ? 0 : clamp64(q.offsets[s], 0, q.tokens);
}
__device__ inline int query_count(const QuerySource& q, int s) {
  const int64_t n = query_begin(q, s + 1) - query_begin(q, s);
  return n < 0 ? 0 : (int)n;
}
// Sequence of a token: the last one that starts at or before it.
__device__ inline int query_seq(const QuerySource& q, int64_t token) {
  if (!q.offsets) return (int)(token / q.per_seq);
  int lo = 0, hi = q.num_seqs;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (query_begin(q, mid) <= token) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// Keys that token j of n sees of its sequence's L rows: those up to its own
// position L - n + j, and the prefix.
__device__ inline int visible_keys(const QuerySource& q, int s, int j, int n, int L) {
  if (q.all || L == 0) return L;
  int v = L - n + j + 1;
  if (q.prefix) v = max(v, min(q.prefix[s], L));
  return max(v, 0);
}
// Query tiles of `rows` tokens: as the key tiles.
__device__ inline int64_t query_tile(const QuerySource& q, int s, int rows) {
  if (q.offsets) return query_begin(q, s) / rows + s;
  return (int64_t)s * ((q.per_seq + rows - 1) / rows);
}
__device__ inline int query_find(const QuerySource& q, int64_t tile, int rows) {
  if (!q.offsets) return (int)(tile / ((q.per_seq + rows - 1) / rows));
  int lo = 0, hi = q.num_seqs;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (query_tile(q, mid, rows) <= tile) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
inline int64_t query_tiles(const QuerySource& q, int rows) {
  return q.offsets ? q.tokens / rows + q.num_seqs + 1 : (int64_t)q.num_seqs * ((q.per_seq + rows - 1) / rows);
}
inline int64_t source_tiles(const RowSource& r) {
  return r.offsets ? r.total_rows / kTileKeys + r.num_seqs
                   : (int64_t)r.num_seqs * ((r.region + kTileKeys - 1) / kTileKeys);
}

// Four consecutive elements of a query tensor of any type, aligned to their 8 or 16 bytes.
__device__ inline void load_q4(const void* base, int dtype, int64_t i, float (&x)[4]) {
  if (dtype == LA_DTYPE_F32) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i);
    const uint32_t w[4] = {v.x & 0xFFFF, v.x >> 16, v.y & 0xFFFF, v.y >> 16};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x[e] = dtype == LA_DTYPE_BF16 ? f_of(w[e] << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)w[e]);
  }
}
inline bool q_vec(const void* base, int dtype, int64_t stride, int64_t head) {
  const uintptr_t align = dtype == LA_DTYPE_F32 ? 16 : 8;
  return reinterpret_cast<uintptr_t>(base) % align == 0 && stride % 4 == 0 && head % 4 == 0;
}

inline bool q_wide(const void* base, int64_t stride, int64_t head) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && stride % 8 == 0 && head % 8 == 0;
}

// A query tile as prompt_kernel takes it, found once per call by gather_kernel:
// binary searches over device offsets in every workgroup were a chain of
// dependent loads at its start.
struct alignas(16) QueryTile {
  int32_t j0;       // its first token within the sequence, < 0: no tokens
  int32_t n, L;     // tokens and rows of the sequence
  int32_t prefix;   // rows that every token sees
  int64_t token0;   // first token of the sequence
  int64_t tile0;    // first key tile of the sequence
};
__device__ inline QueryTile make_query_tile(const QuerySource& q, const RowSource& r, int64_t tile, int rows) {
  const int s = query_find(q, tile, rows);
  const int64_t j0 = (tile - query_tile(q, s, rows)) * rows;
  QueryTile t{};
  t.n = query_count(q, s);
  t.j0 = j0 >= 0 && j0 < t.n ? (int)j0 : -1;
  t.L = source_rows(r, s);
  t.prefix = q.all ? t.L : q.prefix && t.L > 0 ? min(q.prefix[s], t.L) : 0;
  t.token0 = query_begin(q, s);
  t.tile0 = t.L > 0 ? source_tile(r, s) : 0;
  return t;
}
// Keys that token j sees (visible_keys).
__device__ inline int tile_visible(const QueryTile& t, int j) { return t.L == 0 ? 0 : max(max(t.L - t.n + j + 1, t.prefix), 0); }

// Gather + expand: the source's rows as 16-bit latent tiles and rotated rope
// keys (rows_c, rope), then K and V of `heads` heads from row `head0` of the
// weights (16-bit, the tiles' type; kx and vx hold those heads only).
struct ExpandProblem {
  RowSource src;
  int f16;          // 16-bit type: fp16 or bf16
  void* rows_c;     // [tile][64][512]
  void* rope;       // [tile] operand order
  int32_t* tile_rows;  // rows of each tile
  QuerySource q;       // its tiles of query_rows tokens go to q_info (q_tiles = 0: none)
  QueryTile* q_info;
  int64_t q_tiles;
  int query_rows;
  const void* W_UK;
  const void* W_UV;
  void* kx;  // [head][tile] operand order
  void* vx;
  float k_scale;  // times K and the rope keys
  int head0, heads;
};
bool expand_fits(int64_t tiles, int64_t q_tiles);  // one launch of the gather takes them
hipError_t launch_gather(const ExpandProblem& p, hipStream_t stream, int ncu);
hipError_t launch_expand(const ExpandProblem& p, hipStream_t stream, int ncu);
// 16-bit copy of n weights of another type.
hipError_t launch_convert(const void* src, int src_dtype, void* dst, int f16, int64_t n, hipStream_t stream);

// Attention over expanded keys and values.
struct PromptProblem {
  QuerySource q;
  RowSource src;
  int f16;
  const void* kx;
  const void* vx;
  const void* rope;
  const QueryTile* q_info;  // q_tiles of them, or nullptr: one sequence, every token sees every row
  int nh, head0, heads;  // weight heads; this launch's
  float q_scale;  // times the queries (1: the keys are scaled already)
  void* out;  // (tokens, nh, 128) in out_dtype
  int out_dtype;
  int splits;  // > 1: partial sums below, joined by launch_join
  float* part_o;    // [split][token][nh][128], normalised
  float* part_lse;  // [split][token][nh], base 2
  int64_t q_tiles;
  int group;  // order of the workgroups: heads of an XCD taken together (a divisor of heads / 8), or 0
  int nope_vec, rope_vec, table_vec;  // 16-byte (queries: whole-vector) aligned
  int q_wide;  // 16-bit queries: 16-byte aligned
};
int prompt_query_rows();  // query tokens per workgroup
// Most items (query tile, head, key part) of a launch.
constexpr int64_t kMostPromptItems = most_blocks(256) - 8;
hipError_t launch_prompt(const PromptProblem& p, hipStream_t stream);

// Joins partial results of the same (token, head) rows by their log-sum-exps.
constexpr int kJoinSplits = 32;  // at most
struct JoinProblem {
  int64_t rows;  // tokens * nh
  int nh, dv;
  int splits;
  const float* part_o;    // [split][row][dv]
  const float* part_lse;  // [split][row]
  // decode results to join with them: output rows and, for their
  // log-sum-exps, the step whose partial slots they came from (num_seqs 0: none)
  DecodeProblem step[2];
  const float* step_out[2];
  void* out;
  int out_dtype;
};
hipError_t launch_join(const JoinProblem& p, hipStream_t stream);
// The same from the steps' partial slots (step[0] is there; step_out unused):
// merge, W_UV and join in one (la_proj.hip). Both steps hold fp16 slots and
// have 16-bit W_UV.
bool merge_join_supported(const DecodeProblem& p);
hipError_t launch_merge_join(const JoinProblem& j, hipStream_t stream, int ncu);

// Any type and head shape: absorbed queries (fp32), one workgroup per (token, head).
struct GenericPrompt {
  QuerySource q;  // q_nope unused
  RowSource src;
  const float* q_abs;
  const void* W_UV;
  int wuv_dtype;
  int nh, dc, dR, dv;
  float scale_log2;
  void* out;
  int out_dtype;
};
bool generic_prompt_supported(int dc, int dR);
hipError_t launch_generic_prompt(const GenericPrompt& p, hipStream_t stream);

// Queries of the absorbed forms: packed fp32 copies (rotated if asked) and,
// for the decode kernels, every token as a sequence of its own: its visible
// rows and a copy of its sequence's block table (of identity blocks where the
// cache is contiguous).
struct TokenProblem {
  QuerySource q;
  RowSource src;
  int nh, dn, dR;
  float* q_nope;   // (tokens, nh, dn), or nullptr
  float* q_rope;   // (tokens, nh, dR), or nullptr
  int32_t* lens;   // (tokens), or nullptr
  int32_t* table;  // (tokens, blocks_per_seq), entries past used_blocks are never read
  int block_size, blocks_per_seq, used_blocks;
  int vec;  // queries are whole-vector aligned
};
hipError_t launch_tokens(const TokenProblem& p, hipStream_t stream);
// Absorption straight from queries of any type and strides (q.per_seq per
// sequence) into the matrix kernels' operand order (qprep_index), as
// launch_absorb_mfma writes it from packed, rotated fp32 ones.
struct AbsorbQueries {
  QuerySource q;
  RowSource src;       // positions: token j of n of a sequence with L rows is at L - n + j
  const int32_t* pos;  // or given (device, one per token)
  int64_t low;         // > 0: also what the rounded rows leave, in a second array so many elements on
  uint8_t* most;       // fp16 parts of any queries: (rows, kMostRow), exponents of the pieces' largest numbers (fit_f16); or nullptr
};
// A score from its sum. Fused with a subtraction of the same score, rounded (its row's maximum), the product would leave
// its rounding there, past 2^24 more than an exponent: the row's largest weight was infinite.
__device__ inline float scaled_score(float sum, float scale) {
#pragma clang fp contract(off)
  return sum * scale;
}

// Two fp16 parts of a row of queries. Its pieces of 32 latent columns, and its rope part (which comes doubled, for keys in
// halves), are each divided by a power of two that goes by their largest number m (as exponent_of has it): 1 for m from
// 2^-6 on below 2^15, where two parts hold it to 2^-19 or better (and where it is not finite), else the one that brings it to
// 2^14. top_f16 and fit_f16 are those powers' exponents without and with the first case.
constexpr int kMostPieces = 17, kMostRow = 20;
constexpr float kUpRope = 2.f;
__device__ inline int exponent_of(float m) { return (int)(__builtin_bit_cast(uint32_t, m) >> 23); }  // m >= 0
__device__ inline float power_of_2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
__device__ inline int top_f16(int e) { return e == 255 ? 0 : max(e, 27) - 127 - 14; }
__device__ inline int fit_f16(int e) { return e >= 127 - 6 && e < 127 + 15 ? 0 : top_f16(e); }
bool absorb_any_supported(const QuerySource& q, const RowSource& r, const void* W_UK, int w_dtype, const la_mla_config& c);
// out_mode 1: bf16, 2: fp16; zero_out as for launch_absorb_mfma.
hipError_t launch_absorb_any(const AbsorbQueries& x, const void* W_UK, int w_dtype, void* out, int out_mode, float scale,
                             int nh, hipStream_t stream, int ncu, float* zero_out = nullptr, int64_t zero_n = 0);
// fp32 -> out_dtype
hipError_t launch_cast(const float* src, void* dst, int out_dtype, int64_t n, hipStream_t stream);

}  // namespace la
