// Types shared by the draft-tree and cache-cutting kernels (la_tree.hip,
// la_weigh.hip, la_evict.hip) and the C-ABI layer. Not installed.
#pragma once

#include "la_prompt.hpp"

namespace la {

constexpr int kTreeNodes = LA_TREE_MAX_NODES;
static_assert(kTreeNodes == 64, "a node's ancestors are the bits of one word, a tree's nodes the lanes of one wave");

// Trees as the attention kernels take them, and packed fp32 queries, rotated by
// their nodes' positions if asked (launch_tree_queries).
struct TreeQueries {
  QuerySource q;  // offsets nullptr, per_seq nodes
  RowSource src;
  const int32_t* parents;  // (num_seqs, nodes)
  int nh, dn, dR;
  float* q_nope;   // (tokens, nh, dn), or nullptr
  float* q_rope;   // (tokens, nh, dR), or nullptr
  int32_t* lens;   // (num_seqs): rows, 0 where they are fewer than the nodes; with chunks, the plan of the spans behind them (num_seqs + 2)
  int chunks, shortest;  // of spans, and the fewest tiles of one (DecodeProblem); 0: none
  int step;              // tiles that the attention kernel takes at a time: a span has whole ones
  uint64_t* seen;  // TreeStep
  float* cos;
  float* sin;
  int32_t* pos;    // (tokens): the nodes' positions, or nullptr
  int vec;  // queries are whole-vector aligned
};
hipError_t launch_tree_queries(const TreeQueries& p, hipStream_t stream);

// Any type and head shape: absorbed fp32 queries, one workgroup per (token, head).
struct PlainTree {
  RowSource src;  // with TreeQueries' lens
  const uint64_t* seen;
  int nodes;
  const float* q_abs;
  const float* q_rope;  // rotated
  const void* W_UV;
  int wuv_dtype;
  int nh, dc, dR, dv;
  float scale_log2;
  void* out;
  int out_dtype;
};
hipError_t launch_plain_tree(const PlainTree& p, hipStream_t stream);

// A cache whose rows move within their sequences.
struct MovedRows {
  char* kv;
  int64_t row_bytes;
  int64_t total_rows;
  int num_seqs;
  int region;              // rows of a sequence at most (offsets == nullptr)
  const int32_t* offsets;  // device, num_seqs + 1, or nullptr
  int32_t* lens;           // device, num_seqs
  const int32_t* block_table;
  int block_size;
  int blocks_per_seq;
  int64_t pool_blocks;
};
// First row of sequence s in the row space of the sequences, and the rows it has room for.
__device__ inline int64_t moved_begin(const MovedRows& r, int s) {
  return r.offsets ? clamp64(r.offsets[s], 0, r.total_rows) : (int64_t)s * r.region;
}
__device__ inline int moved_room(const MovedRows& r, int s) {
  if (!r.offsets) return r.region;
  return (int)max(clamp64(r.offsets[s + 1], 0, r.total_rows) - moved_begin(r, s), (int64_t)0);
}
// Row of position pos, which lies in the sequence's room (block ids are clamped into the pool).
__device__ inline int64_t moved_index(const MovedRows& r, int s, int64_t begin, int pos) {
  if (!r.block_table) return begin + pos;
  const int64_t b = clamp64(r.block_table[(int64_t)s * r.blocks_per_seq + pos / r.block_size], 0, r.pool_blocks - 1);
  return b * r.block_size + pos % r.block_size;
}
__device__ inline char* moved_row(const MovedRows& r, int s, int64_t begin, int pos) {
  return r.kv + moved_index(r, s, begin, pos) * r.row_bytes;
}
// Between the reads of rows that move and the barrier after which others write there: the
// barrier alone does not wait for loads.
__device__ inline void rows_read() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// The widest accesses that rows and the cache's address allow: 16, 8, 4, 2 or 1 bytes.
inline int moved_unit(const MovedRows& r) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(r.kv) | (uintptr_t)r.row_bytes | 16;
  return (int)(a & -a);
}

// la_accept_kv.
struct AcceptProblem {
  MovedRows rows;
  int nodes;
  const int32_t* path;  // (num_seqs, nodes)
};
hipError_t launch_accept(const AcceptProblem& p, hipStream_t stream);

// la_weigh_kv: packed fp32 queries (q_rope rotated), tokens per sequence.
struct WeighProblem {
  RowSource src;
  int tokens;  // of every sequence
  int nh, dc, dR;
  const float* q_abs;   // (num_seqs * tokens, nh, dc)
  const float* q_rope;  // (num_seqs * tokens, nh, dR)
  float scale_log2;
  float* weights;
  float* sums;  // plain form: (num_seqs * tokens, nh, 2), rows' maxima and what their exponentials' sums divide by
  // matrix form: the queries' operands (qprep_index, weigh_query_scale), what their
  // rounding left `low` elements on, and one piece of the call, `seqs` sequences from seq0 on and of
  // each `count` of its (token, head) rows from row0 on (a multiple of 32)
  int seq0, seqs, row0, count;
  const void* q_prep;
  int64_t low;
  uint8_t* most;  // fp16: the exponents of the operands' pieces (AbsorbQueries)
  int spans;       // workgroups that share the tiles of a row group
  int tiles;       // the piece's at most: `scores` has room for so many (offsets that overlap add up to more rows than there are)
  float* scores;   // [tile][32 rows][32 keys] of `row_blocks` blocks per tile
  float* part;     // [slot][m, l][rows rounded up to 32]
};
hipError_t launch_weigh_plain(const WeighProblem& p, hipStream_t stream);
// The matrix form: 16-bit and FP8 rows of 512 + 64 elements. A piece's workspace goes
// by the tiles (of 32 rows) that its sequences have room for.
bool weigh_mfma_supported(const WeighProblem& p);
constexpr int kWeighKeys = 32, kWeighRows = 4096;  // keys per tile; (token, head) rows of a piece at most
inline bool weigh_f16(int kv_dtype) { return kv_dtype != LA_DTYPE_BF16; }  // the products' type: fp16, or bf16
float weigh_query_scale(const WeighProblem& p);
hipError_t launch_weigh_queries(const WeighProblem& p, hipStream_t stream);  // q_prep from q_abs and q_rope
int weigh_spans(int rows, int ncu);
inline size_t weigh_score_bytes(int64_t tiles, int rows) { return (size_t)tiles * ((rows + 31) / 32) * 4096; }
inline size_t weigh_part_bytes(int spans, int seqs, int rows) {
  return (size_t)(spans + seqs - 1) * 2 * ((rows + 31) / 32 * 32) * sizeof(float);
}
hipError_t launch_weigh_mfma(const WeighProblem& p, hipStream_t stream, int ncu);

// la_evict_kv.
struct EvictProblem {  // from: nullptr where no sequence can have more than `keep` rows
  MovedRows rows;
  float* weights;
  int keep, first, last;
  int32_t* kept;    // (num_seqs, keep)
  int32_t* start;   // (num_seqs): the first position that gets another row, keep if none does
  uint32_t* from;   // (num_seqs, keep): the rows that stay, as rows of the cache
  char* staged;     // evict_staged: (num_seqs, keep) rows; else nullptr
};
// Whether the rows go through a copy of them (few sequences: fewer stripes than compute units).
bool evict_staged(const EvictProblem& p, int ncu);
hipError_t launch_evict(const EvictProblem& p, hipStream_t stream);

}  // namespace la
