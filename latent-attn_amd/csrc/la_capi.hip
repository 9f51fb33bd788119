// extern "C" entry points of liblatent_attn_hip.so (declared in
// include/latent_attn.h): argument checking, split-KV planning, workspace
// carving and kernel dispatch. Host code only; the kernels live in the other
// files: attention in la_mfma.hip (128 heads a workgroup), la_mfma16.hip (16),
// la_f32.hip (float32) and la_generic.hip (any shape), absorption and merge +
// projection for 16-bit weights and the merge for float32 ones in la_proj.hip,
// the other absorption in la_f32.hip and la_generic.hip, la_append.hip,
// la_naive.hip.
#include "la_internal.hpp"
#include "la_prompt.hpp"

#include <algorithm>
#include <cmath>
#include <mutex>
#include <vector>

namespace la {
namespace {

thread_local int g_last_hip_error = 0;

int record_hip(hipError_t e) {
  g_last_hip_error = (int)e;
  return LA_ERROR_HIP;
}

bool valid_dtype(int d) { return d == LA_DTYPE_F32 || d == LA_DTYPE_F16 || d == LA_DTYPE_BF16; }
// latent caches may also be FP8 E4M3 (weights may not)
bool valid_cache_dtype(int d) { return valid_dtype(d) || d == LA_DTYPE_FP8_E4M3; }

// Same conditions as MLAConfig::validate (src/mla_config.cuh:35-40) plus the
// rotate-half requirement of an even rope dimension.
bool valid_cfg(const la_mla_config* c) {
  if (!c) return false;
  if (c->kv_lora_rank <= 0 || c->qk_nope_head_dim <= 0 || c->qk_rope_head_dim <= 0) return false;
  if (c->num_heads <= 0 || c->v_head_dim <= 0) return false;
  return (c->qk_rope_head_dim % 2) == 0;
}

int cu_count() {
  static std::mutex mu;
  static std::vector<int> cache;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  std::lock_guard<std::mutex> lock(mu);
  if ((int)cache.size() <= dev) cache.resize(dev + 1, 0);
  if (cache[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cache[dev] = n;
  }
  return cache[dev];
}

constexpr size_t kAlign = 256;
size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

enum Variant { kAuto = 0, kGeneric = 1, kMfma = 2 };

struct Plan {
  bool mfma = false;
  bool f32 = false;  // decode_f32_kernel
  int waves16 = 0;  // 4 / 8: decode_mfma16_kernel with that many waves; 0: decode_mfma_kernel
  int chunk_len = 0;
  int num_chunks = 0;
  int num_slots = 0;
  bool proj_mfma = false;
  bool proj_f32 = false;
  size_t part_scale_off = 0;
  bool absorb_mfma = false;  // q_nope . W_UK on the MFMA kernel
  bool absorb_f32 = false;   // ... in fp32
  bool absorb_prep = false;  // ... writing the attention kernel's 16-bit Q rows directly
  size_t q_abs_off = 0, q_prep_off = 0, part_o_off = 0, part_lse_off = 0, total = 0;
};

// Fills the problem (without workspace pointers) and the plan. The args'
// chunk_rows / kernel_variant fields are tuning overrides (0 = automatic).
// coarse: the chunks of one 128-head (or VALU) workgroup per target block, also
// for the kernels with 16 heads per workgroup: fewer partial slots, for a caller
// whose scratch does not hold the others.
int prepare(const la_decode_args* a, DecodeProblem* p, Plan* plan, bool coarse = false) {
  if (!a || !valid_cfg(&a->cfg)) return LA_ERROR_INVALID_VALUE;
  const int chunk_rows = a->chunk_rows;
  const int variant = a->kernel_variant;
  if (chunk_rows < 0 || variant < kAuto || variant > kMfma || a->rope_rows < 0) return LA_ERROR_INVALID_VALUE;
  if (a->num_seqs < 0 || a->queries_per_seq < 1 || a->total_rows < 0) return LA_ERROR_INVALID_VALUE;
  if (!valid_cache_dtype(a->kv_dtype) || !valid_dtype(a->w_uv_dtype)) return LA_ERROR_INVALID_VALUE;
  const bool paged = a->block_table != nullptr;
  if (paged) {
    // pool of total_rows rows in blocks; sequences are virtual regions of
    // blocks_per_seq blocks whose filled length comes from seq_lens
    if (a->block_size <= 0 || a->blocks_per_seq <= 0 || a->seq_offsets || !a->seq_lens ||
        a->total_rows % a->block_size != 0 || (int64_t)a->blocks_per_seq * a->block_size > INT32_MAX ||
        a->total_rows > (int64_t)UINT32_MAX ||  // pool rows are 32-bit in the MFMA kernel
        (a->num_seqs > 0 && a->total_rows < a->block_size))  // a pool without a block: nothing to clamp into
      return LA_ERROR_INVALID_VALUE;
  } else if (!a->seq_offsets && (a->seq_len < 0 || (int64_t)a->num_seqs * a->seq_len > a->total_rows)) {
    return LA_ERROR_INVALID_VALUE;
  }
  const bool absorb = a->q_nope != nullptr;
  if (absorb == (a->q_absorbed != nullptr)) return LA_ERROR_INVALID_VALUE;
  if (absorb && (!a->W_UK || !valid_dtype(a->w_uk_dtype))) return LA_ERROR_INVALID_VALUE;
  const la_mla_config& c = a->cfg;

  *p = DecodeProblem{};
  p->kv = a->kv_cache;
  p->kv_dtype = a->kv_dtype;
  p->row_elems = c.kv_lora_rank + c.qk_rope_head_dim;
  p->total_rows = a->total_rows;
  p->num_seqs = a->num_seqs;
  p->seq_len = a->seq_offsets ? 0 : a->seq_len;
  p->offsets = a->seq_offsets;
  p->lens = a->seq_lens;
  if (paged) {
    p->block_table = a->block_table;
    p->block_size = a->block_size;
    p->blocks_per_seq = a->blocks_per_seq;
    p->pool_blocks = a->total_rows / a->block_size;
    p->pool_last = (int)std::min<int64_t>(std::max<int64_t>(p->pool_blocks - 1, 0), INT32_MAX);
    set_tile_divisor(*p, (uint32_t)std::max(a->block_size / 32, 1));
    p->seq_len = a->blocks_per_seq * a->block_size;       // virtual region per sequence
    p->total_rows = (int64_t)a->num_seqs * p->seq_len;    // the virtual row space the plan covers
  }
  p->qps = a->queries_per_seq;
  p->nh = c.num_heads;
  p->Hq = a->queries_per_seq * c.num_heads;
  p->q_abs = a->q_absorbed;
  p->q_rope = a->q_rope;
  p->W_UV = a->W_UV;
  p->wuv_dtype = a->w_uv_dtype;
  p->rope_cos = a->rope_cos;
  p->rope_sin = a->rope_sin;
  p->rope_rows = a->rope_rows;
  p->out = a->output;
  p->dc = c.kv_lora_rank;
  p->dR = c.qk_rope_head_dim;
  p->dv = c.v_head_dim;
  p->scale_log2 = (float)(kLog2e / std::sqrt((double)(c.qk_nope_head_dim + c.qk_rope_head_dim)));

  if (a->num_seqs == 0) {
    *plan = Plan{};
    return LA_SUCCESS;
  }
  if (!a->q_rope || !a->W_UV || !a->rope_cos || !a->rope_sin || !a->output) return LA_ERROR_INVALID_VALUE;
  if (a->total_rows > 0 && !a->kv_cache) return LA_ERROR_INVALID_VALUE;

  Plan pl;
  // the fp32 MFMA kernels write and read 16-byte vectors of the workspace
  const bool ws_aligned = (reinterpret_cast<uintptr_t>(a->workspace) & 15) == 0;
  // An FP8 E4M3 cache runs on the MFMA kernel too (its tiles are expanded to
  // bf16 in LDS); the VALU kernel (kernel_variant 1) reads it as well.
  const bool mfma_ok = mfma_supported(*p);
  if (variant == kMfma && !mfma_ok) return LA_ERROR_NOT_SUPPORTED;
  if (variant == kGeneric || !mfma_ok) {
    if (!generic_supported(*p)) return LA_ERROR_NOT_SUPPORTED;
    pl.mfma = false;
    pl.f32 = variant == kAuto && decode_f32_supported(*p) && ws_aligned;
  } else {
    pl.mfma = true;
  }

  const int64_t total = paged ? p->total_rows : a->seq_offsets ? a->total_rows : (int64_t)a->num_seqs * a->seq_len;
  const int ncu = cu_count();
  // Up to 32 query heads take the 16-head kernel: 128-head workgroups run the
  // matrix work of 128 heads whatever their number (32 x 4099 rows, attention us,
  // 128-head against 16-head workgroups: 16 heads 51 / 33, 32 heads 52 / 38, 64
  // heads 53 / 60). With 17 to 32, two workgroups read each row, and once a
  // 16-bit cache streams from HBM (not from the 256 MB behind the L2s) their
  // shorter tiles in flight fall behind (a step over one sequence: 196,608 rows
  // 78.2 / 76.5, 212,992 81.0 / 86.3, 262,144 93.7 / 105.0; 32 sequences of 163,840
  // in all 66.2 / 51.2, 245,760 89.0 / 86.0, 262,144 92.8 / 93.4; 64 over 327,680
  // 112.8 / 115.1). FP8 rows stay (64 x 8192: 155 / 126), and so do caches cut
  // over their filled rows, whose number only the device knows (64 regions of
  // 8192 rows, a step with 128-head workgroups over the regions and this one:
  // full 164 / 169, three quarters 147 / 152, half 123 / 98, a quarter 118 / 55).
  const int heads16 = pl.mfma ? p->Hq / 16 : 0;
  const bool by_fill = a->seq_lens && chunk_rows == 0 && 4LL * a->num_seqs <= ncu;
  const int64_t most16 = a->num_seqs == 1 ? 200000 : 240000;
  const bool few_heads = pl.mfma && (heads16 == 1 || (heads16 == 2 && (a->kv_dtype == LA_DTYPE_FP8_E4M3 || by_fill ||
                                                                       total <= most16)));
  int64_t L, min_rows = 64;
  if (chunk_rows > 0) {
    L = chunk_rows;
  } else if (pl.f32 && !coarse) {
    // two workgroups per CU, but no chunks under 128 rows while one per CU
    // remains: their partial rows (2 KB per head) cost the merge more than the
    // second workgroup gains (4 x 1000 rows, 128 heads: 51.5 us a step against
    // 53.8 with 64; with 16 heads 43 against 36.5)
    const int64_t groups = (p->Hq + 15) / 16;
    const int64_t chunks = std::max<int64_t>(1, 2LL * ncu / groups);
    L = std::max<int64_t>(((total + chunks - 1) / chunks + 15) / 16 * 16, 64);
    if (L < 128 && groups * ((total + 127) / 128) >= ncu) L = 128;
    min_rows = std::min<int64_t>(L, 128);
  } else if (few_heads && !coarse) {
    // two workgroups per CU and no more (16 heads x 131168 rows: 33.4 us with
    // 257-row chunks, 37 with 128, 35.6 with 513), but one while a sequence has
    // more than 128 chunks: its row's merge reads them all in a few workgroups
    // (16 heads, a step over 1 x 32768 rows 41.4 us with 512 chunks, 29.1 with
    // 256; 1 x 131072 60.6 and 48.1; 3 x 30000 40.7 and, with 384, 37.6; 4 x 32768
    // 45.5 and 43.5; 32 x 4099 46.5 and 49.2); whole tiles only where a paged cache
    // needs them, so that rounding leaves no CU without a chunk
    const int64_t chunks = std::max<int64_t>(std::min(2LL * ncu / heads16, 128LL * a->num_seqs), ncu);
    L = (total + chunks - 1) / chunks;
    L = std::max<int64_t>((L + 15) / 16 * 16, 64);
  } else {
    int64_t groups = pl.mfma ? (p->Hq + mfma_heads_per_group() - 1) / mfma_heads_per_group() : p->Hq;
    int64_t target_blocks = pl.mfma ? ncu : 4LL * ncu;
    int64_t chunks = std::max<int64_t>(1, target_blocks / std::max<int64_t>(1, groups));
    L = (total + chunks - 1) / chunks;
    // MFMA path: each workgroup (one chunk, one group of up to 128 query
    // heads) writes a partial row of dc fp16 values per head; keep them
    // below the bytes the workgroup streams from a 16-bit cache (rows of
    // dc + dR), so short batches (B = 1) do not trade a cheaper attention
    // launch for a merge that reads more than the cache: 128 heads need at
    // least 114 rows (128 after rounding). The floor counts rows, so for an
    // FP8 cache (rows of half the bytes) the partials may reach twice the
    // cache bytes. Head groups share a chunk's rows (several queries over
    // one cache), each writing its own partials, so the floor is per group.
    if (pl.mfma) {
      const int64_t hg = std::min<int64_t>(p->Hq, mfma_heads_per_group());
      const int64_t rows = (hg * c.kv_lora_rank + c.kv_lora_rank + c.qk_rope_head_dim - 1) /
                           (c.kv_lora_rank + c.qk_rope_head_dim);
      L = std::max<int64_t>(L, rows);
      min_rows = std::max<int64_t>((rows + 63) / 64 * 64, 64);
    }
    L = (L + 63) / 64 * 64;
    L = std::max<int64_t>(L, 64);
  }
  if (L > (int64_t)1 << 30) L = (int64_t)1 << 30;
  if ((pl.mfma || pl.f32) && L > kMaxChunkRows) L = kMaxChunkRows;
  if (paged && (pl.mfma || pl.f32)) L = (L + 63) / 64 * 64;  // MFMA tiles start block-aligned
  const int64_t nchunks = total > 0 ? (total + L - 1) / L : 0;
  if (nchunks > (int64_t)1 << 30) return LA_ERROR_INVALID_VALUE;
  pl.chunk_len = (int)L;
  pl.num_chunks = (int)nchunks;
  // More heads take it while its workgroups fill the chip at most twice (the
  // 128-head kernel would have a quarter of the CUs busy): 1 x 512 rows and
  // 128 heads 16.2 us on the 128-head kernel, 7.9 here; 1 x 8192 17.0 / 11.6;
  // four times that (16 queries over 2048 rows) 21.7 / 36.3. With at most one
  // workgroup per CU, 8 waves take 128 positions per round trip.
  if (pl.mfma && (few_heads || (heads16 > 2 && nchunks * heads16 <= 2 * ncu)))
    pl.waves16 = nchunks * heads16 <= ncu && L >= 128 ? 8 : 4;
  pl.num_slots = nchunks > 0 ? (int)(nchunks + a->num_seqs - 1) : 0;

  const int64_t tokens = (int64_t)a->num_seqs * a->queries_per_seq;
  pl.absorb_mfma = absorb && absorb_mfma_supported(a->w_uk_dtype, c.num_heads, c.qk_nope_head_dim, c.kv_lora_rank) &&
                   (reinterpret_cast<uintptr_t>(a->q_nope) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(a->W_UK) & 15) == 0;
  pl.absorb_f32 = absorb && absorb_f32_supported(a->q_nope, a->W_UK, a->w_uk_dtype, static_cast<float*>(a->workspace),
                                                 c.qk_nope_head_dim, c.kv_lora_rank);
  pl.absorb_prep = pl.mfma && pl.absorb_mfma;
  size_t off = 0;
  if (absorb && !pl.absorb_prep) {
    pl.q_abs_off = off;
    off += align_up((size_t)tokens * c.num_heads * c.kv_lora_rank * sizeof(float));
  }
  if (pl.mfma) {
    pl.q_prep_off = off;
    off += align_up((size_t)a->num_seqs * qprep_rows_per_seq(p->Hq) * kQPrepRow * 2);
  }
  // the MFMA kernel writes its partial rows as scaled fp16, the VALU kernel as fp32
  p->part_f16 = pl.mfma ? 1 : 0;
  pl.part_o_off = off;
  off += align_up((size_t)pl.num_slots * p->Hq * c.kv_lora_rank * (pl.mfma ? 2 : 4));
  if (pl.mfma) {
    pl.part_scale_off = off;  // two per row (column halves), then part_m: one per row
    off += align_up((size_t)pl.num_slots * p->Hq * 3 * sizeof(float));
  }
  pl.part_lse_off = off;
  const int piece = (int)std::min<int64_t>((min_rows + 31) / 32 * 32, L);  // shortest piece of filled rows
  const bool filled = a->seq_lens && chunk_rows == 0 && (pl.mfma || pl.f32) && 4LL * a->num_seqs <= nchunks &&
                      total <= INT32_MAX && (L > piece || a->seq_offsets || p->seq_len % L != 0) &&
                      piece_rows((uint32_t)total, (uint32_t)(nchunks - a->num_seqs), piece) <= kMaxChunkRows;
  off += align_up((size_t)pl.num_slots * p->Hq * sizeof(float));
  pl.proj_mfma = project_mfma_supported(*p);
  pl.proj_f32 = project_f32_supported(*p) && ws_aligned;
  pl.total = off;

  p->chunk_len = pl.chunk_len;
  // Per-sequence lengths: the chunks are pieces of the sequences' filled rows
  // (seq_in_plan), down to the plan's shortest chunk, while there are four or
  // more per sequence (100 sequences of 100 to 4000 rows over 256 chunks, too
  // uneven pieces: 165 us a step against 147 over their 4096-row regions; 64 of
  // 300 to 8192: 120 against 154; 32 of 500 to 8000 in 32768-row regions: 74
  // against 208), and unless the regions' chunks are already of that length and
  // end with their regions: the pieces would be the same ones, found again on
  // the device (32 of 100 to 500 rows in 512-row regions, 128 heads: 36.4 against
  // 35.5, fp8 38.5 against 37.1).
  if (filled) p->chunk_len = -piece;
  p->num_chunks = pl.num_chunks;
  p->num_slots = pl.num_slots;
  *plan = pl;
  return LA_SUCCESS;
}

// The latent-half merge: few query rows leave most CUs idle in the full-row
// merge, so it is split over the two latent halves, which add into the
// output (zeroed first by the kernel that writes the attention kernel's
// 16-bit queries: the absorb kernel, or prep_q when the queries come
// absorbed and there is at least one chunk; where the attention kernel takes
// the fp32 queries itself, by that one).
bool merge_halves(const DecodeProblem& p, const Plan& plan) {
  const bool zeroed = plan.f32 ? plan.num_chunks > 0  // by decode_f32_kernel itself
                               : plan.mfma && (plan.absorb_prep || plan.num_chunks > 0);
  return zeroed && (plan.proj_f32 || (plan.proj_mfma && plan.mfma)) && merge_project_blocks(p) < cu_count();
}

// ev_b / ev_e (optional) are recorded around the attention kernel, which runs
// max(repeat, 1) times between them. tail (optional): what a kernel that reads
// the step's partial slots next takes from it and leaves to it.
struct StepTail {
  DecodeProblem p;               // out: the problem with its slots' addresses
  bool merge = true;             // false: the slots stay as they are, nothing is written to the output
  const void* q_prep = nullptr;  // the same queries' 16-bit rows in a layout that is this step's too
};
int run(const la_decode_args* a, hipStream_t stream, hipEvent_t ev_b = nullptr, hipEvent_t ev_e = nullptr,
        int repeat = 1, bool coarse = false, StepTail* tail = nullptr) {
  if (repeat < 0) return LA_ERROR_INVALID_VALUE;
  DecodeProblem p;
  Plan plan;
  int st = prepare(a, &p, &plan, coarse);
  if (st != LA_SUCCESS) return st;
  if (a->num_seqs == 0) return LA_SUCCESS;

  char* ws = static_cast<char*>(a->workspace);
  bool owned = false;
  if (plan.total > 0) {
    if (ws) {
      if (a->workspace_bytes < plan.total) return LA_ERROR_WORKSPACE;
    } else {
      void* m = nullptr;
      hipError_t e = hipMallocAsync(&m, plan.total, stream);
      if (e != hipSuccess) return record_hip(e);
      ws = static_cast<char*>(m);
      owned = true;
    }
  }
  auto finish = [&](hipError_t e) -> int {
    if (owned) {
      hipError_t f = hipFreeAsync(ws, stream);
      if (e == hipSuccess) e = f;
    }
    return e == hipSuccess ? (int)LA_SUCCESS : record_hip(e);
  };

  const la_mla_config& c = a->cfg;
  const int64_t tokens = (int64_t)a->num_seqs * a->queries_per_seq;
  if (plan.mfma) p.q_prep = ws + plan.q_prep_off;
  // Few query rows leave most CUs idle in the full-row merge: split it over
  // the two latent halves, which add into the output. The kernel that writes
  // the attention kernel's 16-bit queries (the absorb kernel, or prep_q when
  // the queries come absorbed) runs first and zeroes the output.
  const bool merge_halves = (!tail || tail->merge) && la::merge_halves(p, plan);
  float* const zero_out = merge_halves ? a->output : nullptr;
  const int64_t zero_n = merge_halves ? tokens * c.num_heads * c.v_head_dim : 0;
  if (tail && tail->q_prep && plan.absorb_prep) {
    p.q_prep = const_cast<void*>(tail->q_prep);
  } else if (a->q_nope) {
    hipError_t e = hipSuccess;
    if (plan.absorb_prep) {
      // absorbed, scaled 16-bit Q rows for the attention kernel in one pass
      // q_prep in the MFMAs' 16-bit type: fp16 for an fp16 cache, bf16 otherwise
      e = launch_absorb_mfma(a->q_nope, a->W_UK, a->w_uk_dtype, p.q_prep, p.kv_dtype == LA_DTYPE_F16 ? 2 : 1,
                             a->q_rope, p.scale_log2, c.qk_rope_head_dim, (int)tokens, c.num_heads,
                             c.qk_nope_head_dim, c.kv_lora_rank, a->queries_per_seq, stream, zero_out, zero_n);
    } else {
      float* qa = reinterpret_cast<float*>(ws + plan.q_abs_off);
      if (plan.absorb_f32)
        e = launch_absorb_f32(a->q_nope, a->W_UK, qa, (int)tokens, c.num_heads, c.qk_nope_head_dim, c.kv_lora_rank, stream);
      else if (plan.absorb_mfma)
        e = launch_absorb_mfma(a->q_nope, a->W_UK, a->w_uk_dtype, qa, 0, nullptr, 1.f, 0, (int)tokens, c.num_heads,
                               c.qk_nope_head_dim, c.kv_lora_rank, 1, stream);
      else
        e = launch_absorb(a->q_nope, a->W_UK, a->w_uk_dtype, qa, (int)tokens, c.num_heads, c.qk_nope_head_dim,
                          c.kv_lora_rank, stream);
      p.q_abs = qa;
    }
    if (e != hipSuccess) return finish(e);
  }
  p.part_o = reinterpret_cast<float*>(ws + plan.part_o_off);
  p.part_lse = reinterpret_cast<float*>(ws + plan.part_lse_off);
  p.part_scale = plan.mfma ? reinterpret_cast<float*>(ws + plan.part_scale_off) : nullptr;
  p.part_m = plan.mfma ? p.part_scale + (size_t)plan.num_slots * p.Hq * 2 : nullptr;
  if (plan.num_chunks > 0) {
    if (plan.waves16 == 8 && !plan.absorb_prep) {
      p.q_prep = nullptr;  // decode_mfma16_kernel takes the fp32 queries and zeroes the output
    } else if (plan.mfma && !plan.absorb_prep) {
      hipError_t e = launch_prep_q(p, stream, zero_out, zero_n);
      if (e != hipSuccess) return finish(e);
    }
    // the optional events bracket the attention kernel alone
    hipError_t e = hipSuccess;
    const int reps = repeat > 1 ? repeat : 1;
    auto launch_mfma = [&](hipEvent_t b, hipEvent_t en) {
      return plan.waves16 ? launch_decode_mfma16(p, plan.waves16, stream, p.q_prep ? nullptr : zero_out, zero_n, b, en)
                          : launch_decode_mfma(p, stream, b, en);
    };
    if (plan.mfma && reps == 1) {
      e = launch_mfma(ev_b, ev_e);  // recorded by the launch itself
    } else {
      if (ev_b) e = hipEventRecord(ev_b, stream);
      for (int r = 0; r < reps && e == hipSuccess; ++r)
        e = plan.mfma  ? launch_mfma(nullptr, nullptr)
            : plan.f32 ? launch_decode_f32(p, stream, zero_out, zero_n)
                       : launch_decode_generic(p, stream);
      if (e == hipSuccess && ev_e) e = hipEventRecord(ev_e, stream);
    }
    if (e != hipSuccess) return finish(e);
  }
  if (tail) tail->p = p;
  if (tail && !tail->merge) return finish(hipSuccess);
  if (plan.proj_f32) return finish(launch_combine_project_f32(p, stream, merge_halves));
  if (plan.proj_mfma) return finish(launch_combine_project_mfma(p, stream, merge_halves, cu_count()));
  return finish(launch_combine_project(p, stream));
}

la_decode_args shared_cache_args(const void* kv_cache, int kv_dtype, int seq_len, int batch, const float* q_absorbed,
                                 const float* q_rope, const void* W_UV, int w_uv_dtype, const float* rope_cos,
                                 const float* rope_sin, float* output, const la_mla_config* cfg, void* workspace,
                                 size_t workspace_bytes) {
  la_decode_args a{};
  a.rope_rows = seq_len;
  a.kv_cache = kv_cache;
  a.kv_dtype = kv_dtype;
  a.total_rows = seq_len;
  a.num_seqs = 1;
  a.seq_len = seq_len;
  a.seq_offsets = nullptr;
  a.queries_per_seq = batch;
  a.q_absorbed = q_absorbed;
  a.q_rope = q_rope;
  a.W_UV = W_UV;
  a.w_uv_dtype = w_uv_dtype;
  a.rope_cos = rope_cos;
  a.rope_sin = rope_sin;
  a.output = output;
  if (cfg) a.cfg = *cfg;
  a.workspace = workspace;
  a.workspace_bytes = workspace_bytes;
  return a;
}

// Scratch of la_mla_decode_noalloc: one array per GPU, in the code object,
// held until the process ends. Host code never uses the array's name as an
// address (on the host it is only a stand-in for the device symbol): the
// device address comes from hipGetSymbolAddress, once per device, with that
// device current, and is kept per device.
constexpr size_t kNoAllocScratchBytes = (size_t)64 << 20;
constexpr int kMaxDevices = 64;
std::mutex g_scratch_mu;
void* g_scratch_ptr[kMaxDevices] = {};

}  // namespace

static __device__ __align__(256) char scratch[kNoAllocScratchBytes];

namespace {

// The current device's scratch address (looked up on its first use there).
int scratch_ptr(void** out) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return record_hip(e);
  if (dev < 0 || dev >= kMaxDevices) return LA_ERROR_NOT_SUPPORTED;
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void* ptr = nullptr;
    e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
    if (e != hipSuccess) return record_hip(e);
    if (!ptr) return LA_ERROR_HIP;
    g_scratch_ptr[dev] = ptr;
  }
  *out = g_scratch_ptr[dev];
  return LA_SUCCESS;
}

// ---- prompts and shared prefixes ----------------------------------------------------------------------

bool tables_aligned(const RowSource& r) {
  return ((reinterpret_cast<uintptr_t>(r.cos) | reinterpret_cast<uintptr_t>(r.sin)) & 15) == 0;
}
// Parts that the keys of `tiles` tiles are cut into when `blocks` workgroups
// would run: one workgroup per CU, down to two tiles each, and two per CU where
// each keeps 16 tiles (partial rows cost a workgroup and the join as much as
// several tiles; a step of 32 tokens over 16 heads x 8192 shared rows 50 us with
// 32 parts, 46 with 16; 64 tokens over 128 heads 177 with 4, 183 with 2).
int key_splits(int64_t blocks, int64_t tiles, int least) {
  const int64_t ncu = cu_count();
  const int64_t two = (2 * ncu + blocks - 1) / blocks, one = (ncu + blocks - 1) / blocks;
  const int64_t n = tiles >= 16 * two ? two : std::min(one, tiles / 2);
  return (int)std::max<int64_t>(least, std::min<int64_t>(n, 32));
}
// Heads of an XCD that prompt_kernel takes together: as many as fill its CUs'
// two workgroups each, four at least (their keys and values share its L2, and
// the long query tiles of several heads do not end the call); with all 16 of
// 128 heads / 8 / 4 / one after another, a call, us: 300 rows 42.4 / 46.1 / 46.4 /
// 47.5, 600 78.1 / 72.5 / 75.2 / 83.1, 1001 113 / 110 / 115 / 122, 2000 273 / 274 /
// 268 / 280, 4000 811 / 798 / 795 / 819, 16 x 300 431 / 431 / 431 / 455, 8192 3019 /
// 2782 / 2644 / 2679; 16 heads, both / one: 2000 rows 68.9 / 73.7, 8000 339 / 346.
// 0: heads that the XCDs do not share evenly, in order.
int head_order(int heads, int64_t blocks) {
  if (heads % 8 != 0) return 0;
  const int64_t most = std::max<int64_t>(4, 64 / blocks);
  int group = 1;
  for (int g = 2; g <= heads / 8 && g <= most; ++g)
    if (heads / 8 % g == 0) group = g;
  return group;
}
bool valid_out(int d) { return valid_dtype(d); }
// Head shape of the expanded form's kernels.
bool expanded_dims(const la_mla_config& c) {
  return c.kv_lora_rank == 512 && c.qk_nope_head_dim == 128 && c.qk_rope_head_dim == 64 && c.v_head_dim == 128;
}
bool sixteen_bit(int d) { return d == LA_DTYPE_F16 || d == LA_DTYPE_BF16; }

// Cuts a workspace into 256-byte aligned pieces; with a null base it only counts.
struct Carve {
  char* base;
  size_t at = 0;
  explicit Carve(void* ws) : base(reinterpret_cast<char*>(align_up(reinterpret_cast<uintptr_t>(ws)))) {}
  void* take(size_t bytes) {
    void* const p = base ? base + at : nullptr;
    at += align_up(bytes);
    return p;
  }
  size_t total() const { return at > 0 ? at + kAlign : 0; }  // the base may have to be aligned
};

// The caller's workspace, or one of `need` bytes taken and returned in the order
// of the stream. Under capture it has to be the caller's: whatever replays the
// graph then owns the memory that its kernels write.
struct Scratch {
  void* ws;
  bool owned = false;
  int status = LA_SUCCESS;
  hipStream_t stream;
  Scratch(void* given, size_t given_bytes, size_t need, hipStream_t st) : ws(given), stream(st) {
    if (need == 0) return;
    if (ws) {
      if (given_bytes < need) status = LA_ERROR_WORKSPACE;
    } else {
      hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
      hipError_t e = st ? hipStreamIsCapturing(st, &capture) : hipSuccess;  // (the default stream is never captured)
      if (e == hipSuccess && capture != hipStreamCaptureStatusNone) {
        status = LA_ERROR_WORKSPACE;
        return;
      }
      if (e == hipSuccess) e = hipMallocAsync(&ws, need, st);
      if (e != hipSuccess) status = record_hip(e);
      else owned = true;
    }
  }
  int finish(int st) {
    if (!owned) return st;
    const hipError_t f = hipFreeAsync(ws, stream);
    return st == LA_SUCCESS && f != hipSuccess ? record_hip(f) : st;
  }
};
int status_of(hipError_t e) { return e == hipSuccess ? (int)LA_SUCCESS : record_hip(e); }

// Weights as the expanded form's products take them: 16-bit values of its
// type, from 16-byte aligned rows; others are copied first.
bool weight_as_is(const void* w, int dtype, int f16) {
  return dtype == (f16 ? LA_DTYPE_F16 : LA_DTYPE_BF16) && (reinterpret_cast<uintptr_t>(w) & 15) == 0;
}

// Gather and expansion of `heads` heads at a time, shared by prompts and prefixes.
struct ExpandPlan {
  ExpandProblem p{};
  void* uk_copy = nullptr;
  void* uv_copy = nullptr;
  size_t copy_elems = 0;
};
void carve_expand(Carve& c, ExpandPlan& e, const void* W_UK, int uk_dtype, const void* W_UV, int uv_dtype, int nh) {
  const size_t tiles = (size_t)e.p.src.num_tiles;
  e.p.rows_c = c.take(tiles * kTileCBytes);
  e.p.tile_rows = static_cast<int32_t*>(c.take(tiles * sizeof(int32_t)));
  e.copy_elems = (size_t)nh * 128 * 512;
  e.uk_copy = e.uv_copy = nullptr;
  e.p.W_UK = W_UK;
  e.p.W_UV = W_UV;
  if (!weight_as_is(W_UK, uk_dtype, e.p.f16)) e.p.W_UK = e.uk_copy = c.take(e.copy_elems * 2);
  if (!weight_as_is(W_UV, uv_dtype, e.p.f16)) e.p.W_UV = e.uv_copy = c.take(e.copy_elems * 2);
}
hipError_t start_expand(const ExpandPlan& e, const void* W_UK, int uk_dtype, const void* W_UV, int uv_dtype, bool copy_uk,
                        bool copy_uv, hipStream_t stream) {
  hipError_t r = launch_gather(e.p, stream, cu_count());
  if (r == hipSuccess && copy_uk) r = launch_convert(W_UK, uk_dtype, e.uk_copy, e.p.f16, (int64_t)e.copy_elems, stream);
  if (r == hipSuccess && copy_uv) r = launch_convert(W_UV, uv_dtype, e.uv_copy, e.p.f16, (int64_t)e.copy_elems, stream);
  return r;
}

enum PrefillForm { kPrefillNone = 0, kPrefillPlain = 1, kPrefillExpanded = 2, kPrefillAbsorbed = 3 };

// Expanded keys and values of one launch at most (heads go in groups of it).
constexpr size_t kMaxExpanded = (size_t)8 << 30;

struct Prefill {
  PrefillForm form = kPrefillNone;
  QuerySource q{};
  RowSource src{};
  int block_size = 0, blocks_per_seq = 0, used_blocks = 0;  // of the absorbed form
  int64_t pool_rows = 0;
  bool nope_as_is = false, rope_as_is = false;  // queries that the other forms' kernels take where they lie
  int splits = 1, group = 0;  // of the expanded form: key parts, heads at a time
  int64_t q_tiles = 0;
};

// The decode step of the absorbed form: every token a sequence with its own visible rows.
la_decode_args token_step(const la_prefill_args* a, const Prefill& p, const float* q_nope, const float* q_rope,
                          const int32_t* lens, const int32_t* table, float* out, void* ws, size_t ws_bytes) {
  la_decode_args d{};
  d.kv_cache = a->kv_cache;
  d.kv_dtype = a->kv_dtype;
  d.total_rows = p.pool_rows;
  d.num_seqs = (int32_t)a->tokens;
  d.queries_per_seq = 1;
  d.q_nope = q_nope;
  d.q_rope = q_rope;
  d.W_UK = a->W_UK;
  d.w_uk_dtype = a->w_uk_dtype;
  d.W_UV = a->W_UV;
  d.w_uv_dtype = a->w_uv_dtype;
  d.rope_cos = a->rope_cos;
  d.rope_sin = a->rope_sin;
  d.rope_rows = a->rope_rows;
  d.output = out;
  d.cfg = a->cfg;
  d.seq_lens = lens;
  d.block_table = table;
  d.block_size = p.block_size;
  d.blocks_per_seq = p.blocks_per_seq;
  d.workspace = ws;
  d.workspace_bytes = ws_bytes;
  return d;
}

int prepare_prefill(const la_prefill_args* a, Prefill* out) {
  if (!a || !valid_cfg(&a->cfg) || !valid_cache_dtype(a->kv_dtype) || !valid_dtype(a->w_uk_dtype) ||
      !valid_dtype(a->w_uv_dtype) || !valid_dtype(a->q_dtype) || !valid_out(a->out_dtype))
    return LA_ERROR_INVALID_VALUE;
  const la_mla_config& c = a->cfg;
  if (a->num_seqs < 0 || a->tokens < 0 || a->total_rows < 0 || a->rope_rows < 0 || a->max_seq_rows < 0 ||
      a->kernel_variant < 0 || a->kernel_variant > kPrefillAbsorbed || (a->rotate_q != 0 && a->rotate_q != 1))
    return LA_ERROR_INVALID_VALUE;
  if (a->num_seqs == INT32_MAX || a->tokens > INT32_MAX / c.num_heads) return LA_ERROR_INVALID_VALUE;
  if (a->q_nope_token_stride < 0 || a->q_nope_head_stride < 0 || a->q_rope_token_stride < 0 || a->q_rope_head_stride < 0)
    return LA_ERROR_INVALID_VALUE;
  const bool paged = a->block_table != nullptr;
  if (paged) {
    if (a->block_size <= 0 || a->blocks_per_seq <= 0 || a->seq_offsets || !a->seq_lens ||
        a->total_rows % a->block_size != 0 || (int64_t)a->blocks_per_seq * a->block_size > INT32_MAX ||
        a->total_rows > (int64_t)UINT32_MAX || (a->num_seqs > 0 && a->total_rows < a->block_size))
      return LA_ERROR_INVALID_VALUE;
  } else if (a->seq_offsets) {
    if (a->max_seq_rows != 0 || a->total_rows > INT32_MAX) return LA_ERROR_INVALID_VALUE;
  } else if (a->seq_len < 0 || (int64_t)a->num_seqs * a->seq_len > a->total_rows) {
    return LA_ERROR_INVALID_VALUE;
  }
  Prefill p;
  p.form = kPrefillNone;
  if (a->tokens == 0) {
    *out = p;
    return LA_SUCCESS;
  }
  if (a->num_seqs == 0 || (!a->q_offsets && a->tokens % a->num_seqs != 0)) return LA_ERROR_INVALID_VALUE;
  if (!a->q_nope || !a->q_rope || !a->W_UK || !a->W_UV || !a->rope_cos || !a->rope_sin || !a->output ||
      (a->total_rows > 0 && !a->kv_cache))
    return LA_ERROR_INVALID_VALUE;

  RowSource& r = p.src;
  r.kv = a->kv_cache;
  r.kv_dtype = a->kv_dtype;
  r.row_elems = c.kv_lora_rank + c.qk_rope_head_dim;
  r.total_rows = a->total_rows;
  r.num_seqs = a->num_seqs;
  r.offsets = a->seq_offsets;
  r.lens = a->seq_lens;
  r.cos = a->rope_cos;
  r.sin = a->rope_sin;
  r.rope_rows = a->rope_rows;
  if (paged) {
    r.block_table = a->block_table;
    r.block_size = a->block_size;
    r.blocks_per_seq = a->blocks_per_seq;
    r.pool_blocks = a->total_rows / a->block_size;
    r.region = a->blocks_per_seq * a->block_size;
  } else if (!a->seq_offsets) {
    r.region = r.stride_rows = a->seq_len;
  }
  if (!a->seq_offsets && a->max_seq_rows > 0) r.region = std::min(r.region, a->max_seq_rows);
  r.num_tiles = source_tiles(r);

  QuerySource& q = p.q;
  q.q_nope = a->q_nope;
  q.q_rope = a->q_rope;
  q.dtype = a->q_dtype;
  const bool nope_packed = a->q_nope_token_stride == 0 && a->q_nope_head_stride == 0;
  const bool rope_packed = a->q_rope_token_stride == 0 && a->q_rope_head_stride == 0;
  q.nope_stride = nope_packed ? (int64_t)c.num_heads * c.qk_nope_head_dim : a->q_nope_token_stride;
  q.nope_head = nope_packed ? c.qk_nope_head_dim : a->q_nope_head_stride;
  q.rope_stride = rope_packed ? (int64_t)c.num_heads * c.qk_rope_head_dim : a->q_rope_token_stride;
  q.rope_head = rope_packed ? c.qk_rope_head_dim : a->q_rope_head_stride;
  q.rotate = a->rotate_q;
  q.tokens = a->tokens;
  q.num_seqs = a->num_seqs;
  q.offsets = a->q_offsets;
  q.per_seq = a->q_offsets ? 0 : (int)(a->tokens / a->num_seqs);
  q.prefix = a->prefix_lens;
  // (those that are not aligned are copied: a step over them would run on the VALU)
  const auto as_is = [&](const void* base, int64_t stride, int64_t head, int dim) {
    return a->q_dtype == LA_DTYPE_F32 && head == dim && stride == (int64_t)c.num_heads * dim &&
           (reinterpret_cast<uintptr_t>(base) & 15) == 0;
  };
  p.nope_as_is = as_is(q.q_nope, q.nope_stride, q.nope_head, c.qk_nope_head_dim);
  p.rope_as_is = !a->rotate_q && as_is(q.q_rope, q.rope_stride, q.rope_head, c.qk_rope_head_dim);

  const int64_t q_tiles = query_tiles(q, prompt_query_rows());
  const bool expanded_ok = expanded_dims(c) && (sixteen_bit(a->kv_dtype) || a->kv_dtype == LA_DTYPE_FP8_E4M3) &&
                           device_is_gfx950() && (reinterpret_cast<uintptr_t>(a->output) & 15) == 0 &&
                           r.num_tiles <= INT32_MAX / 128 && expand_fits(r.num_tiles, q_tiles) &&
                           q_tiles <= kMostPromptItems;
  // The absorbed form's block tables: the cache's own, or identity blocks of equal regions.
  if (paged) {
    p.block_size = a->block_size;
    p.pool_rows = a->total_rows;
  } else if (!a->seq_offsets && a->seq_len > 0) {
    p.block_size = a->seq_len % 64 == 0 ? 64 : a->seq_len % 32 == 0 ? 32 : a->seq_len;
    p.pool_rows = (int64_t)a->num_seqs * a->seq_len;
  }
  bool absorbed_ok = p.block_size > 0 && r.region > 0 && p.pool_rows <= (int64_t)UINT32_MAX;  // as la_mla_decode takes
  if (absorbed_ok) {
    p.blocks_per_seq = p.used_blocks = (r.region + p.block_size - 1) / p.block_size;
    absorbed_ok = a->tokens * p.blocks_per_seq <= INT32_MAX &&
                  (int64_t)p.blocks_per_seq * p.block_size <= INT32_MAX;
  }
  // The token step's plan, with aligned addresses in place of what lies in the
  // workspace then.
  alignas(256) static const char any[256] = {0};
  float* const f = reinterpret_cast<float*>(const_cast<char*>(any));
  const int32_t* const ids = reinterpret_cast<const int32_t*>(any);
  DecodeProblem step;
  Plan plan;
  const auto plan_step = [&] {
    const la_decode_args d = token_step(a, p, f, f, ids, ids, f, nullptr, 0);
    return prepare(&d, &step, &plan) == LA_SUCCESS;
  };
  absorbed_ok = absorbed_ok && plan_step();
  const bool plain_ok = generic_prompt_supported(c.kv_lora_rank, c.qk_rope_head_dim);
  if (a->kernel_variant == kPrefillAbsorbed && !absorbed_ok) return LA_ERROR_NOT_SUPPORTED;
  if (a->kernel_variant == kPrefillExpanded && !expanded_ok) return LA_ERROR_NOT_SUPPORTED;
  if (a->kernel_variant == kPrefillPlain && !plain_ok) return LA_ERROR_NOT_SUPPORTED;
  if (a->kernel_variant != 0) {
    p.form = (PrefillForm)a->kernel_variant;
  } else if (expanded_ok) {
    // Microseconds of both forms: launches, then absorption and projection per
    // (token, head) and 1088 products per pair of a token and a row, or expansion
    // per (row, head) and 320 products per pair (a query tile's worth at least).
    // Measured (absorbed / expanded, 128 heads): 1 x 16 of 1000 rows 48 / 76, 64 of
    // 1000 76 / 75, 128 of 1000 111 / 76, 128 of 8192 318 / 475, 200 of 8192 540 /
    // 560, 16 x 16 of 2000 256 / 1900; 16 heads, 17 of 100 28 / 23. Where the step
    // has no matrix kernel (pages or regions that are no multiple of 32 rows, heads
    // no multiple of 16, an unaligned cache) the VALU's takes 0.8 ns per pair and
    // head, and the expanded form, whose gather takes any of these, is faster but
    // for a head or two of one token (its workgroups of a head share an XCD, so
    // fewer than 8 heads cost what 8 do): 128 heads, 16-row pages, 1 x 4 of 2000
    // rows 780 / 109, 16 x 4 9180 / 1610, 1 x 128 of 8192 100,400 / 448; regions of
    // 1000 rows, 1 token 122 / 64; 8 heads, 16 x 4 of 2000 848 / 126, 1 x 64 of 8192
    // 3121 / 58, 1 token of 200 49 / 23, of 131,072 853 / 540; 1 head, 1 token of
    // 32,768 101 / 154, of 131,072 189 / 386, 16 x 4 of 2000 144 / 137.
    const double heads = c.num_heads, seqs = a->num_seqs, n = (double)a->tokens / seqs, rows = std::max(r.region, 1);
    const double absorbed_us = absorbed_ok && plan.mfma ? 27. + a->tokens * heads * (2e-3 + 2.3e-6 * rows)
                                                        : 45. + a->tokens * heads * 8e-4 * rows;
    const double expanded_us = 20. + 1.2 * ((c.num_heads + 7) / 8 * 8) * seqs * rows * (3.1e-4 + 7e-7 * std::max(n, 64.));
    p.form = absorbed_ok && absorbed_us < expanded_us ? kPrefillAbsorbed : kPrefillExpanded;
  } else if (absorbed_ok) {
    p.form = kPrefillAbsorbed;
  } else if (plain_ok) {
    p.form = kPrefillPlain;
  } else {
    return LA_ERROR_NOT_SUPPORTED;
  }

  if (p.form == kPrefillAbsorbed) {
    // The decode plan cuts filled rows where it has four chunks per sequence,
    // which the rounding of its chunks can miss by little (16 x 4 tokens over 500
    // to 6000 rows: 251 chunks for 64 sequences; attention 99.5 us over the
    // regions): longer regions, whose further blocks are never read, reach it.
    bool filled = step.chunk_len < 0;
    for (int more = 1; more < 8 && !filled && a->tokens <= cu_count() / 2; ++more) {
      p.blocks_per_seq = p.used_blocks + more;
      if (a->tokens * p.blocks_per_seq > INT32_MAX || (int64_t)p.blocks_per_seq * p.block_size > INT32_MAX) break;
      filled = plan_step() && step.chunk_len < 0;
    }
    if (!filled) p.blocks_per_seq = p.used_blocks;
  }
  if (p.form == kPrefillExpanded) {
    const size_t head_bytes = (size_t)r.num_tiles * kTileKBytes * 2;
    p.group = (int)std::min<size_t>(c.num_heads, std::max<size_t>(1, head_bytes ? kMaxExpanded / head_bytes : c.num_heads));
    p.q_tiles = q_tiles;
    const int64_t tiles = a->seq_offsets ? a->total_rows / a->num_seqs / kTileKeys + 1 : r.num_tiles / a->num_seqs;
    p.splits = key_splits(p.q_tiles * p.group, tiles, 1);
    // (parts only where there are few items)
    p.group = (int)std::min<int64_t>(p.group, kMostPromptItems / (p.splits * p.q_tiles));
  }
  *out = p;
  return LA_SUCCESS;
}

// Runs the call, or with run = false counts its workspace into *need.
int prefill(const la_prefill_args* a, void* stream_v, bool run_it, size_t* need) {
  const hipStream_t stream = static_cast<hipStream_t>(stream_v);
  Prefill p;
  const int st = prepare_prefill(a, &p);
  if (st != LA_SUCCESS) return st;
  if (need) *need = 0;
  if (p.form == kPrefillNone) return LA_SUCCESS;
  const la_mla_config& c = a->cfg;
  const int nh = c.num_heads;
  const float scale_log2 = (float)(kLog2e / std::sqrt((double)(c.qk_nope_head_dim + c.qk_rope_head_dim)));
  const int64_t rows = a->tokens * nh;

  // the layout is the same whether counted or carved
  ExpandPlan e;
  e.p.src = p.src;
  e.p.f16 = a->kv_dtype == LA_DTYPE_F16;
  float *part_o = nullptr, *part_lse = nullptr, *q_nope = nullptr, *q_rope = nullptr, *q_abs = nullptr, *out32 = nullptr;
  int32_t *lens = nullptr, *table = nullptr;
  void* step_ws = nullptr;
  size_t step_bytes = 0;
  bool cast_merge = false;
  const bool nope_as_is = p.nope_as_is, rope_as_is = p.rope_as_is;
  auto carve = [&](void* ws) {
    Carve v(ws);
    if (p.form == kPrefillExpanded) {
      carve_expand(v, e, a->W_UK, a->w_uk_dtype, a->W_UV, a->w_uv_dtype, nh);
      const size_t tiles = (size_t)p.src.num_tiles;
      e.p.q_info = static_cast<QueryTile*>(v.take((size_t)p.q_tiles * sizeof(QueryTile)));
      e.p.rope = v.take(tiles * kTileRBytes);
      e.p.kx = v.take(tiles * p.group * kTileKBytes);
      e.p.vx = v.take(tiles * p.group * kTileKBytes);
      if (p.splits > 1) {
        part_o = static_cast<float*>(v.take((size_t)p.splits * rows * 128 * sizeof(float)));
        part_lse = static_cast<float*>(v.take((size_t)p.splits * rows * sizeof(float)));
      }
    } else {
      if (!nope_as_is) q_nope = static_cast<float*>(v.take((size_t)rows * c.qk_nope_head_dim * sizeof(float)));
      if (p.form == kPrefillPlain) {
        q_abs = static_cast<float*>(v.take((size_t)rows * c.kv_lora_rank * sizeof(float)));
      } else {
        if (!rope_as_is) q_rope = static_cast<float*>(v.take((size_t)rows * c.qk_rope_head_dim * sizeof(float)));
        lens = static_cast<int32_t*>(v.take((size_t)a->tokens * sizeof(int32_t)));
        table = static_cast<int32_t*>(v.take((size_t)a->tokens * p.blocks_per_seq * sizeof(int32_t)));
        // (the addresses are those of a workspace of any base: only their alignment matters to the plan)
        alignas(256) static const char any[256] = {0};
        const float* f = reinterpret_cast<const float*>(any);
        const la_decode_args d =
            token_step(a, p, nope_as_is ? static_cast<const float*>(a->q_nope) : f,
                       rope_as_is ? static_cast<const float*>(a->q_rope) : f, reinterpret_cast<const int32_t*>(any),
                       reinterpret_cast<const int32_t*>(any), const_cast<float*>(f), nullptr, 0);
        step_bytes = la_mla_decode_workspace_size(&d);
        step_ws = v.take(step_bytes);
        DecodeProblem step;
        Plan plan;
        // The merge that ends the step writes 16-bit rows itself (the step's own merge and a cast / so: 16 x 4 tokens x
        // 128 heads 119 / 109 us a call, 16 x 8 112 / 94, 2 x 2 33.0 / 30.9, 1 token 33.2 / 31.3)
        cast_merge = a->out_dtype != LA_DTYPE_F32 && prepare(&d, &step, &plan) == LA_SUCCESS && merge_join_supported(step);
        if (a->out_dtype != LA_DTYPE_F32 && !cast_merge)
          out32 = static_cast<float*>(v.take((size_t)rows * c.v_head_dim * sizeof(float)));
      }
    }
    return v.total();
  };
  const size_t total = carve(nullptr);
  if (p.form == kPrefillAbsorbed && step_bytes == 0) return LA_ERROR_NOT_SUPPORTED;
  if (need) *need = total;
  if (!run_it) return LA_SUCCESS;
  Scratch scratch(a->workspace, a->workspace_bytes, total, stream);
  if (scratch.status != LA_SUCCESS) return scratch.status;
  carve(scratch.ws);

  if (p.form == kPrefillExpanded) {
    e.p.q = p.q;
    e.p.q_tiles = p.q_tiles;
    e.p.query_rows = prompt_query_rows();
    e.p.k_scale = scale_log2;  // the softmax's scale goes into the keys before their one rounding
    e.p.heads = p.group;
    hipError_t r = start_expand(e, a->W_UK, a->w_uk_dtype, a->W_UV, a->w_uv_dtype, e.uk_copy, e.uv_copy, stream);
    PromptProblem m{};
    m.q = p.q;
    m.src = p.src;
    m.f16 = e.p.f16;
    m.kx = e.p.kx;
    m.vx = e.p.vx;
    m.rope = e.p.rope;
    m.q_info = e.p.q_info;
    m.nh = nh;
    m.q_scale = 1.f;
    m.out = a->output;
    m.out_dtype = a->out_dtype;
    m.splits = p.splits;
    m.part_o = part_o;
    m.part_lse = part_lse;
    m.q_tiles = p.q_tiles;
    m.nope_vec = q_vec(p.q.q_nope, p.q.dtype, p.q.nope_stride, p.q.nope_head);
    m.rope_vec = q_vec(p.q.q_rope, p.q.dtype, p.q.rope_stride, p.q.rope_head);
    m.q_wide = q_wide(p.q.q_nope, p.q.nope_stride, p.q.nope_head) && q_wide(p.q.q_rope, p.q.rope_stride, p.q.rope_head);
    m.table_vec = tables_aligned(p.src);
    for (int h = 0; h < nh && r == hipSuccess; h += p.group) {
      e.p.head0 = m.head0 = h;
      e.p.heads = m.heads = std::min(p.group, nh - h);
      m.group = head_order(m.heads, (a->tokens + prompt_query_rows() - 1) / prompt_query_rows() * m.splits);
      r = launch_expand(e.p, stream, cu_count());
      if (r == hipSuccess) r = launch_prompt(m, stream);
    }
    if (r == hipSuccess && p.splits > 1) {
      JoinProblem j{};
      j.rows = rows;
      j.nh = nh;
      j.dv = 128;
      j.splits = p.splits;
      j.part_o = part_o;
      j.part_lse = part_lse;
      j.out = a->output;
      j.out_dtype = a->out_dtype;
      r = launch_join(j, stream);
    }
    return scratch.finish(status_of(r));
  }

  TokenProblem t{};
  t.q = p.q;
  t.src = p.src;
  t.nh = nh;
  t.dn = c.qk_nope_head_dim;
  t.dR = c.qk_rope_head_dim;
  t.q_nope = q_nope;
  t.q_rope = q_rope;
  t.lens = lens;
  t.table = table;
  t.block_size = p.block_size;
  t.blocks_per_seq = p.blocks_per_seq;
  t.used_blocks = p.used_blocks;
  t.vec = q_vec(p.q.q_nope, p.q.dtype, p.q.nope_stride, p.q.nope_head) && q_vec(p.q.q_rope, p.q.dtype, p.q.rope_stride, p.q.rope_head);
  const float* const qn = nope_as_is ? static_cast<const float*>(a->q_nope) : q_nope;
  if (p.form == kPrefillPlain) {
    hipError_t r = q_nope ? launch_tokens(t, stream) : hipSuccess;
    if (r != hipSuccess) return scratch.finish(record_hip(r));
    const int s2 = la_absorb_q(qn, a->W_UK, a->w_uk_dtype, q_abs, (int)a->tokens, &c, stream_v);
    if (s2 != LA_SUCCESS) return scratch.finish(s2);
    GenericPrompt g{};
    g.q = p.q;
    g.src = p.src;
    g.q_abs = q_abs;
    g.W_UV = a->W_UV;
    g.wuv_dtype = a->w_uv_dtype;
    g.nh = nh;
    g.dc = c.kv_lora_rank;
    g.dR = c.qk_rope_head_dim;
    g.dv = c.v_head_dim;
    g.scale_log2 = scale_log2;
    g.out = a->output;
    g.out_dtype = a->out_dtype;
    return scratch.finish(status_of(launch_generic_prompt(g, stream)));
  }
  hipError_t r = launch_tokens(t, stream);
  if (r != hipSuccess) return scratch.finish(record_hip(r));
  float* const out = out32 ? out32 : static_cast<float*>(a->output);  // (cast_merge: the step leaves it alone)
  const la_decode_args d = token_step(a, p, qn, rope_as_is ? static_cast<const float*>(a->q_rope) : q_rope, lens, table,
                                      out, step_ws, step_bytes);
  StepTail tail;
  tail.merge = !cast_merge;
  int s3 = run(&d, stream, nullptr, nullptr, 1, false, &tail);
  if (s3 == LA_SUCCESS && cast_merge) {
    JoinProblem j{};
    j.rows = rows;
    j.nh = nh;
    j.dv = c.v_head_dim;
    j.step[0] = tail.p;
    j.out = a->output;
    j.out_dtype = a->out_dtype;
    s3 = status_of(launch_merge_join(j, stream, cu_count()));
  }
  if (s3 == LA_SUCCESS && out32) s3 = status_of(launch_cast(out32, a->output, a->out_dtype, rows * c.v_head_dim, stream));
  return scratch.finish(s3);
}

// ---- a prefix, expanded once --------------------------------------------------------------------------

RowSource prefix_source(const void* rows, int dtype, int n, const la_mla_config& c, const float* cos, const float* sin,
                        int64_t rope_rows) {
  RowSource r{};
  r.kv = rows;
  r.kv_dtype = dtype;
  r.row_elems = c.kv_lora_rank + c.qk_rope_head_dim;
  r.total_rows = n;
  r.num_seqs = 1;
  r.region = r.stride_rows = n;
  r.cos = cos;
  r.sin = sin;
  r.rope_rows = rope_rows;
  r.num_tiles = source_tiles(r);
  return r;
}

int expand(const la_expand_args* a, hipStream_t stream, bool run_it, size_t* need) {
  if (!a || !valid_cfg(&a->cfg) || !valid_cache_dtype(a->kv_dtype) || !valid_dtype(a->w_uk_dtype) ||
      !valid_dtype(a->w_uv_dtype) || a->rows < 0 || a->rope_rows < 0)
    return LA_ERROR_INVALID_VALUE;
  if (need) *need = 0;
  if (!expanded_dims(a->cfg) || a->kv_dtype == LA_DTYPE_F32) return LA_ERROR_NOT_SUPPORTED;
  if (a->rows == 0) return LA_SUCCESS;
  if (!a->kv_cache || !a->W_UK || !a->W_UV || !a->rope_cos || !a->rope_sin) return LA_ERROR_INVALID_VALUE;
  ExpandPlan e;
  e.p.src = prefix_source(a->kv_cache, a->kv_dtype, a->rows, a->cfg, a->rope_cos, a->rope_sin, a->rope_rows);
  if (!expand_fits(e.p.src.num_tiles, 0)) return LA_ERROR_NOT_SUPPORTED;
  e.p.f16 = a->kv_dtype == LA_DTYPE_F16;
  auto carve = [&](void* ws) {
    Carve v(ws);
    carve_expand(v, e, a->W_UK, a->w_uk_dtype, a->W_UV, a->w_uv_dtype, a->cfg.num_heads);
    return v.total();
  };
  const size_t total = carve(nullptr);
  if (need) *need = total;
  if (!run_it) return LA_SUCCESS;
  if (!a->expanded || (reinterpret_cast<uintptr_t>(a->expanded) & (kAlign - 1)) != 0 ||
      a->expanded_bytes < la_expanded_size(a->rows, &a->cfg))
    return LA_ERROR_INVALID_VALUE;
  if (!device_is_gfx950()) return LA_ERROR_NOT_SUPPORTED;
  Scratch scratch(a->workspace, a->workspace_bytes, total, stream);
  if (scratch.status != LA_SUCCESS) return scratch.status;
  carve(scratch.ws);
  const size_t kv = (size_t)a->cfg.num_heads * e.p.src.num_tiles * kTileKBytes;
  e.p.kx = a->expanded;
  e.p.vx = static_cast<char*>(a->expanded) + kv;
  e.p.rope = static_cast<char*>(a->expanded) + 2 * kv;
  e.p.k_scale = 1.f;
  e.p.head0 = 0;
  e.p.heads = a->cfg.num_heads;
  hipError_t r = start_expand(e, a->W_UK, a->w_uk_dtype, a->W_UV, a->w_uv_dtype, e.uk_copy, e.uv_copy, stream);
  if (r == hipSuccess) r = launch_expand(e.p, stream, cu_count());
  return scratch.finish(status_of(r));
}

// ---- decode behind a shared prefix --------------------------------------------------------------------

int decode_shared(const la_shared_args* a, hipStream_t stream, bool run_it, size_t* need) {
  if (!a || !valid_cfg(&a->own.cfg)) return LA_ERROR_INVALID_VALUE;
  const la_mla_config& c = a->own.cfg;
  const int nh = c.num_heads;
  if (!valid_out(a->out_dtype) || a->prefix_len < 0 || a->kernel_variant < 0 || a->kernel_variant > 2 ||
      a->own.num_seqs < 0 || a->own.queries_per_seq < 1 || a->own.q_absorbed || a->own.rope_rows < 0)
    return LA_ERROR_INVALID_VALUE;
  const int64_t tokens = (int64_t)a->own.num_seqs * a->own.queries_per_seq;
  if (tokens > INT32_MAX / nh) return LA_ERROR_INVALID_VALUE;
  if (need) *need = 0;
  if (tokens == 0) return LA_SUCCESS;
  if (!a->own.q_nope || !a->own.q_rope || !a->output || !a->own.rope_cos || !a->own.rope_sin || !a->own.W_UK ||
      !a->own.W_UV || (a->prefix_len > 0 && !a->prefix))
    return LA_ERROR_INVALID_VALUE;
  const int P = a->prefix_len;
  const int64_t half = c.qk_rope_head_dim / 2;

  la_decode_args own = a->own;
  // own rows start at position P; tables that end before it give their last row, as everywhere
  const int64_t first = own.rope_rows > 0 ? std::min<int64_t>(P, own.rope_rows - 1) : P;
  own.rope_cos += first * half;
  own.rope_sin += first * half;
  if (own.rope_rows > 0) own.rope_rows -= first;
  own.chunk_rows = own.kernel_variant = 0;
  own.workspace = nullptr;
  own.workspace_bytes = 0;
  alignas(256) static const char any[256] = {0};  // stands for an aligned address while sizes are counted
  own.output = reinterpret_cast<float*>(const_cast<char*>(any));

  const bool expanded_ok = a->expanded && (reinterpret_cast<uintptr_t>(a->expanded) & (kAlign - 1)) == 0 &&
                           expanded_dims(c) && own.kv_dtype != LA_DTYPE_F32 && device_is_gfx950();
  if (a->kernel_variant == 2 && !expanded_ok) return LA_ERROR_NOT_SUPPORTED;
  // Microseconds beside the own rows': over latent rows 1.75e-6 per (token, head,
  // row) and 5 to 27 of launches (a second attention and its slots); over the
  // expanded form its bytes at 5 TB/s. A step over latent rows / expanded: 128
  // heads, 8192 rows with 16, 32, 48, 64 tokens 75 / 126, 112 / 134, 162 / 154,
  // 196 / 159; 2000 rows with 8, 16, 32 51 / 59, 53 / 54, 68 / 58; 500 rows with 1,
  // 4, 16 33 / 36, 41 / 44, 41 / 39; 16 heads, 512 rows with 2 32 / 28; 8192 with
  // 1, 8, 32 36 / 39, 41 / 38, 56 / 42; 32768 with 8, 32, 100 61 / 73, 76 / 78,
  // 157 / 110. Where the latent rows have no matrix kernel (query heads of all
  // tokens no multiple of 16, unaligned rows), always the expanded form: 8 heads, 1
  // behind 64 rows 85 / 50, behind 32768 279 / 104; 17 heads, 2 behind 4000 225 / 84,
  // 8 behind 32768 3480 / 151.
  la_decode_args pre{};
  DecodeProblem pre_step;
  Plan pre_plan;
  int pre_st = LA_SUCCESS;
  if (P > 0) {
    pre = a->own;
    pre.kv_cache = a->prefix;
    pre.total_rows = pre.seq_len = P;
    pre.num_seqs = 1;
    pre.queries_per_seq = (int32_t)tokens;
    pre.seq_offsets = pre.seq_lens = pre.block_table = nullptr;
    pre.block_size = pre.blocks_per_seq = 0;
    pre.chunk_rows = pre.kernel_variant = 0;
    pre.workspace = nullptr;
    pre.workspace_bytes = 0;
    pre.output = own.output;
    pre_st = prepare(&pre, &pre_step, &pre_plan);
  }
  const double pairs = (double)nh * P, all = pairs * tokens;
  const bool expanded =
      P > 0 && expanded_ok &&
      (a->kernel_variant == 2 ||
       (a->kernel_variant == 0 && (pre_st != LA_SUCCESS || !pre_plan.mfma ||
                                   pairs * 512. / 5e6 < std::min(27., 5. + 4e-6 * all) + 1.75e-6 * all)));

  PromptProblem m{};
  size_t pre_bytes = 0;
  if (expanded) {
    pre.num_seqs = 0;
    m.src = prefix_source(a->prefix, own.kv_dtype, P, c, a->own.rope_cos, a->own.rope_sin, a->own.rope_rows);
    m.q.q_nope = own.q_nope;
    m.q.q_rope = own.q_rope;
    m.q.dtype = LA_DTYPE_F32;
    m.q.nope_head = c.qk_nope_head_dim;
    m.q.nope_stride = (int64_t)nh * c.qk_nope_head_dim;
    m.q.rope_head = c.qk_rope_head_dim;
    m.q.rope_stride = (int64_t)nh * c.qk_rope_head_dim;
    m.q.tokens = tokens;
    m.q.num_seqs = 1;
    m.q.per_seq = (int)tokens;
    m.q.all = 1;
    m.f16 = own.kv_dtype == LA_DTYPE_F16;
    m.nh = m.heads = nh;
    m.q_scale = (float)(kLog2e / std::sqrt((double)(c.qk_nope_head_dim + c.qk_rope_head_dim)));
    m.out_dtype = LA_DTYPE_F32;
    m.q_tiles = query_tiles(m.q, prompt_query_rows());
    m.nope_vec = q_vec(m.q.q_nope, m.q.dtype, m.q.nope_stride, m.q.nope_head);
    m.rope_vec = q_vec(m.q.q_rope, m.q.dtype, m.q.rope_stride, m.q.rope_head);
    m.table_vec = tables_aligned(m.src);
    m.splits = key_splits(m.q_tiles * nh, m.src.num_tiles, 2);  // 2: a join follows either way
    if (m.q_tiles * nh * m.splits > kMostPromptItems) return LA_ERROR_NOT_SUPPORTED;
  } else if (pre_st != LA_SUCCESS) {
    return pre_st;
  }
  // Validates the own rows' step. One kernel merges their slots, projects and joins
  // where the slots are the MFMA kernels'. Heads in whole blocks of 32 query rows
  // lie alike in both steps, which then share the absorbed queries (steps that
  // merge by themselves do not: their absorption zeroes the output of a half-row merge).
  DecodeProblem own_step;
  Plan own_plan;
  int st = prepare(&own, &own_step, &own_plan);
  if (st != LA_SUCCESS) return st;
  bool one = P > 0 && merge_join_supported(own_step), share = nh % 32 == 0 && own_plan.absorb_prep;
  if (pre.num_seqs > 0) {
    one = one && merge_join_supported(pre_step);
    share = share && one && pre_plan.absorb_prep;
  }
  const size_t own_bytes = la_mla_decode_workspace_size(&own);
  if (pre.num_seqs > 0) pre_bytes = la_mla_decode_workspace_size(&pre);

  const int64_t rows = tokens * nh;
  void *own_ws = nullptr, *pre_ws = nullptr;
  float *own_out = nullptr, *pre_out = nullptr;
  auto carve = [&](void* ws) {
    Carve v(ws);
    own_ws = v.take(own_bytes);
    if (!one) own_out = static_cast<float*>(v.take((size_t)rows * c.v_head_dim * sizeof(float)));
    if (expanded) {
      m.part_o = static_cast<float*>(v.take((size_t)m.splits * rows * 128 * sizeof(float)));
      m.part_lse = static_cast<float*>(v.take((size_t)m.splits * rows * sizeof(float)));
    } else if (P > 0) {
      pre_ws = v.take(pre_bytes);
      if (!one) pre_out = static_cast<float*>(v.take((size_t)rows * c.v_head_dim * sizeof(float)));
    }
    return v.total();
  };
  const size_t total = carve(nullptr);
  if (need) *need = total;
  if (!run_it) return LA_SUCCESS;
  Scratch scratch(a->workspace, a->workspace_bytes, total, stream);
  if (scratch.status != LA_SUCCESS) return scratch.status;
  carve(scratch.ws);
  JoinProblem j{};
  j.rows = rows;
  j.nh = nh;
  j.dv = c.v_head_dim;
  j.out = a->output;
  j.out_dtype = a->out_dtype;
  if (expanded) {
    const size_t kv = (size_t)nh * m.src.num_tiles * kTileKBytes;
    m.kx = a->expanded;
    m.vx = static_cast<const char*>(a->expanded) + kv;
    m.rope = static_cast<const char*>(a->expanded) + 2 * kv;
    st = status_of(launch_prompt(m, stream));
    j.splits = m.splits;
    j.part_o = m.part_o;
    j.part_lse = m.part_lse;
  } else if (P > 0) {
    if (!one) pre.output = pre_out;
    pre.workspace = pre_ws;
    pre.workspace_bytes = pre_bytes;
    StepTail tail;
    tail.merge = !one;
    st = run(&pre, stream, nullptr, nullptr, 1, false, &tail);
    j.step[1] = tail.p;
    j.step_out[1] = pre_out;
  }
  if (st == LA_SUCCESS) {
    if (!one) own.output = own_out;
    own.workspace = own_ws;
    own.workspace_bytes = own_bytes;
    StepTail tail;
    tail.merge = !one;
    if (share && !expanded && P > 0) tail.q_prep = j.step[1].q_prep;
    st = run(&own, stream, nullptr, nullptr, 1, false, &tail);
    j.step[0] = tail.p;
    j.step_out[0] = own_out;
  }
  if (st == LA_SUCCESS) st = status_of(one ? launch_merge_join(j, stream, cu_count()) : launch_join(j, stream));
  return scratch.finish(st);
}

}  // namespace
}  // namespace la

extern "C" {

const char* la_status_string(int status) {
  switch (status) {
    case LA_SUCCESS: return "success";
    case LA_ERROR_INVALID_VALUE: return "invalid value";
    case LA_ERROR_NOT_SUPPORTED: return "not supported";
    case LA_ERROR_WORKSPACE: return "workspace too small";
    case LA_ERROR_HIP: return "HIP runtime error";
    default: return "unknown status";
  }
}

int la_last_hip_error(void) { return la::g_last_hip_error; }

int la_abi_version(void) { return LA_ABI_VERSION; }

size_t la_mla_decode_workspace_size(const la_decode_args* args) {
  la::DecodeProblem p;
  la::Plan plan;
  if (la::prepare(args, &p, &plan) != LA_SUCCESS) return 0;
  size_t bytes = plan.total;
  if (args->num_seqs > 0 && args->kv_dtype == LA_DTYPE_F32 && args->kernel_variant == la::kAuto) {
    // Alignment alone decides between the two float32 kernels, and either may
    // take more chunks (one head over 100,000 rows: 782 on the VALU kernel, 481
    // on the fp32 MFMA kernel): the size serves both, so it does not depend on
    // the pointers that the step is called with.
    la_decode_args a = *args;
    a.kernel_variant = la::kGeneric;
    if (la::prepare(&a, &p, &plan) == LA_SUCCESS) bytes = std::max(bytes, plan.total);
    alignas(16) static const float aligned[4] = {0.f};
    a.kernel_variant = la::kAuto;
    a.workspace = nullptr;
    a.kv_cache = a.q_rope = a.rope_cos = a.rope_sin = aligned;
    if (a.q_absorbed) a.q_absorbed = aligned;
    if (la::prepare(&a, &p, &plan) == LA_SUCCESS) bytes = std::max(bytes, plan.total);
  }
  return bytes;
}

static_assert(sizeof(la_plan_info) == 32 + sizeof(size_t) && offsetof(la_plan_info, workspace_bytes) == 32,
              "the layout of callers built against seven 32-bit fields");
int la_mla_decode_plan(const la_decode_args* args, la_plan_info* info) {
  if (!info) return LA_ERROR_INVALID_VALUE;
  la::DecodeProblem p;
  la::Plan plan;
  const int st = la::prepare(args, &p, &plan);
  if (st != LA_SUCCESS) return st;
  *info = la_plan_info{};
  info->workspace_bytes = la_mla_decode_workspace_size(args);
  if (args->num_seqs == 0) return LA_SUCCESS;
  info->attention = plan.mfma ? LA_PLAN_ATTENTION_MFMA : plan.f32 ? LA_PLAN_ATTENTION_MFMA_F32 : LA_PLAN_ATTENTION_VALU;
  info->chunk_rows = plan.chunk_len;
  info->num_chunks = plan.num_chunks;
  info->num_slots = plan.num_slots;
  const int group = plan.mfma ? la::mfma_heads_per_group() : plan.f32 ? 16 : 1;
  info->head_groups = (p.Hq + group - 1) / group;
  info->heads_per_workgroup = (int16_t)(plan.waves16 ? 16 : group);
  info->filled_rows = p.chunk_len < 0;
  if (plan.proj_f32) info->merge = la::merge_halves(p, plan) ? LA_PLAN_MERGE_MFMA_F32_HALVES : LA_PLAN_MERGE_MFMA_F32;
  else if (!plan.proj_mfma) info->merge = LA_PLAN_MERGE_VALU;
  else info->merge = la::merge_halves(p, plan) ? LA_PLAN_MERGE_MFMA_HALVES : LA_PLAN_MERGE_MFMA;
  if (!args->q_nope) info->absorb = LA_PLAN_ABSORB_NONE;
  else if (plan.absorb_prep) info->absorb = LA_PLAN_ABSORB_MFMA_QPREP;
  else if (plan.absorb_f32) info->absorb = LA_PLAN_ABSORB_MFMA_F32;
  else info->absorb = plan.absorb_mfma ? LA_PLAN_ABSORB_MFMA : LA_PLAN_ABSORB_VALU;
  return LA_SUCCESS;
}

int la_mla_decode(const la_decode_args* args, void* stream) { return la::run(args, static_cast<hipStream_t>(stream)); }

int la_mla_decode_profiled(const la_decode_args* args, void* stream, void* event_begin, void* event_end,
                           int32_t repeat) {
  return la::run(args, static_cast<hipStream_t>(stream), static_cast<hipEvent_t>(event_begin),
                 static_cast<hipEvent_t>(event_end), repeat);
}

int la_stream_ceiling(const la_decode_args* args, int32_t ring, void* stream, void* event_begin, void* event_end,
                      int32_t repeat) {
  if (ring != 3 && ring != 4 || repeat < 0) return LA_ERROR_INVALID_VALUE;
  la::DecodeProblem p;
  la::Plan plan;
  const int st = la::prepare(args, &p, &plan);
  if (st != LA_SUCCESS) return st;
  if (!plan.mfma || p.block_table || (p.kv_dtype != LA_DTYPE_BF16 && p.kv_dtype != LA_DTYPE_F16))
    return LA_ERROR_NOT_SUPPORTED;
  if (plan.num_chunks == 0) return LA_SUCCESS;
  p.chunk_len = plan.chunk_len;  // the copies walk the regions
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e = hipSuccess;
  if (event_begin) e = hipEventRecord(static_cast<hipEvent_t>(event_begin), s);
  for (int r = 0; r < (repeat > 1 ? repeat : 1) && e == hipSuccess; ++r) e = la::launch_stream_copies(p, ring, s);
  if (e == hipSuccess && event_end) e = hipEventRecord(static_cast<hipEvent_t>(event_end), s);
  return e == hipSuccess ? (int)LA_SUCCESS : la::record_hip(e);
}

int la_mla_decode_noalloc(const la_decode_args* args, void* stream) {
  la::DecodeProblem p;
  la::Plan plan;
  int st = la::prepare(args, &p, &plan);
  const bool coarse = st == LA_SUCCESS && plan.total > la::kNoAllocScratchBytes;
  if (coarse) st = la::prepare(args, &p, &plan, true);
  if (st != LA_SUCCESS) return st;
  if (plan.total > la::kNoAllocScratchBytes) return LA_ERROR_WORKSPACE;
  la_decode_args a = *args;
  a.workspace = nullptr;
  a.workspace_bytes = la::kNoAllocScratchBytes;
  if (plan.total > 0) {
    const int sp = la::scratch_ptr(&a.workspace);
    if (sp != LA_SUCCESS) return sp;
  }  // else: no workspace is needed and none is passed
  return la::run(&a, static_cast<hipStream_t>(stream), nullptr, nullptr, 1, coarse);
}

size_t la_mla_decode_noalloc_max_bytes(void) { return la::kNoAllocScratchBytes; }

int la_fused_mla(const void* kv_cache, int kv_dtype, int seq_len, const float* q_absorbed, const float* q_rope,
                 const void* W_UV, int w_uv_dtype, const float* rope_cos, const float* rope_sin, float* output,
                 const la_mla_config* cfg, void* workspace, size_t workspace_bytes, void* stream) {
  if (!cfg || seq_len < 0 || !q_absorbed) return LA_ERROR_INVALID_VALUE;
  la_decode_args a = la::shared_cache_args(kv_cache, kv_dtype, seq_len, 1, q_absorbed, q_rope, W_UV, w_uv_dtype,
                                           rope_cos, rope_sin, output, cfg, workspace, workspace_bytes);
  return la::run(&a, static_cast<hipStream_t>(stream));
}

int la_batched_fused_mla(const void* kv_cache, int kv_dtype, int seq_len, int batch_size, const float* q_absorbed,
                         const float* q_rope, const void* W_UV, int w_uv_dtype, const float* rope_cos,
                         const float* rope_sin, float* output, const la_mla_config* cfg, void* workspace,
                         size_t workspace_bytes, void* stream) {
  if (!cfg || seq_len < 0 || batch_size <= 0 || !q_absorbed) return LA_ERROR_INVALID_VALUE;
  la_decode_args a = la::shared_cache_args(kv_cache, kv_dtype, seq_len, batch_size, q_absorbed, q_rope, W_UV,
                                           w_uv_dtype, rope_cos, rope_sin, output, cfg, workspace, workspace_bytes);
  return la::run(&a, static_cast<hipStream_t>(stream));
}

size_t la_fused_mla_workspace_size_dt(int seq_len, int batch_size, const la_mla_config* cfg, int kv_dtype,
                                      int w_uv_dtype) {
  if (!cfg || seq_len < 0 || batch_size <= 0) return 0;
  // Only plan-relevant fields are read. Which kernel family runs also depends
  // on pointer alignment, so return the largest of the families' plans (the
  // fp32 MFMA kernel has no variant of its own: 0 plans it).
  alignas(256) static const char dummy[256] = {0};
  const float* d = reinterpret_cast<const float*>(dummy);
  size_t best = 0;
  for (int variant : {0, 1, 2}) {
    la_decode_args a = la::shared_cache_args(dummy, kv_dtype, seq_len, batch_size, d, d, dummy, w_uv_dtype, d, d,
                                             const_cast<float*>(d), cfg, nullptr, 0);
    a.kernel_variant = variant;
    la::DecodeProblem p;
    la::Plan plan;
    if (la::prepare(&a, &p, &plan) == LA_SUCCESS && plan.total > best) best = plan.total;
  }
  return best;
}

size_t la_fused_mla_workspace_size(int seq_len, int batch_size, const la_mla_config* cfg) {
  // every cache dtype with every weight dtype
  size_t best = 0;
  for (int kv : {LA_DTYPE_F16, LA_DTYPE_BF16, LA_DTYPE_F32, LA_DTYPE_FP8_E4M3})
    for (int w : {LA_DTYPE_F16, LA_DTYPE_BF16, LA_DTYPE_F32})
      best = std::max(best, la_fused_mla_workspace_size_dt(seq_len, batch_size, cfg, kv, w));
  return best;
}

size_t la_naive_mla_workspace_size(int seq_len, const la_mla_config* cfg) {
  if (!la::valid_cfg(cfg) || seq_len < 0) return 0;
  return la::naive_workspace_bytes(seq_len, cfg->num_heads, cfg->qk_nope_head_dim, cfg->v_head_dim);
}

int la_naive_mla(const void* kv_cache, int kv_dtype, int seq_len, const void* W_UK, int w_uk_dtype, const void* W_UV,
                 int w_uv_dtype, const float* q_nope, const float* q_rope, const float* rope_cos,
                 const float* rope_sin, float* output, const la_mla_config* cfg, void* workspace,
                 size_t workspace_bytes, void* stream) {
  if (!la::valid_cfg(cfg) || seq_len < 0 || !la::valid_cache_dtype(kv_dtype) || !la::valid_dtype(w_uk_dtype) ||
      !la::valid_dtype(w_uv_dtype))
    return LA_ERROR_INVALID_VALUE;
  if (!W_UK || !W_UV || !q_nope || !q_rope || !rope_cos || !rope_sin || !output || (seq_len > 0 && !kv_cache))
    return LA_ERROR_INVALID_VALUE;
  const size_t need = la::naive_workspace_bytes(seq_len, cfg->num_heads, cfg->qk_nope_head_dim, cfg->v_head_dim);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  la::NaiveProblem p{};
  p.kv = kv_cache;
  p.kv_dtype = kv_dtype;
  p.S = seq_len;
  p.W_UK = W_UK;
  p.wuk_dtype = w_uk_dtype;
  p.W_UV = W_UV;
  p.wuv_dtype = w_uv_dtype;
  p.q_nope = q_nope;
  p.q_rope = q_rope;
  p.rope_cos = rope_cos;
  p.rope_sin = rope_sin;
  p.rope_rows = seq_len;  // the reference indexes cos/sin by position < seq_len (src/fused_mla.cu:158-159)
  p.out = output;
  p.nh = cfg->num_heads;
  p.dn = cfg->qk_nope_head_dim;
  p.dR = cfg->qk_rope_head_dim;
  p.dc = cfg->kv_lora_rank;
  p.dv = cfg->v_head_dim;
  p.scale = (float)(1.0 / std::sqrt((double)(cfg->qk_nope_head_dim + cfg->qk_rope_head_dim)));
  void* ws = workspace;
  bool owned = false;
  if (ws) {
    if (workspace_bytes < need) return LA_ERROR_WORKSPACE;
  } else if (need > 0) {
    hipError_t e = hipMallocAsync(&ws, need, st);
    if (e != hipSuccess) return la::record_hip(e);
    owned = true;
  }
  hipError_t e = la::launch_naive(p, ws, st);
  if (owned) {
    hipError_t f = hipFreeAsync(ws, st);
    if (e == hipSuccess) e = f;
  }
  return e == hipSuccess ? (int)LA_SUCCESS : la::record_hip(e);
}

int la_append_kv(const la_append_args* a, void* stream) {
  if (!a || !la::valid_cfg(&a->cfg) || !la::valid_cache_dtype(a->kv_dtype) || !la::valid_cache_dtype(a->src_dtype))
    return LA_ERROR_INVALID_VALUE;
  if (a->num_seqs < 0 || a->tokens_per_seq < 0 || a->total_rows < 0 || a->rope_rows < 0) return LA_ERROR_INVALID_VALUE;
  const bool paged = a->block_table != nullptr;
  if (paged) {
    if (a->block_size <= 0 || a->blocks_per_seq <= 0 || a->seq_offsets || a->total_rows % a->block_size != 0 ||
        (a->num_seqs > 0 && a->total_rows < a->block_size))  // a pool without a block: nothing to clamp into
      return LA_ERROR_INVALID_VALUE;
  } else if (!a->seq_offsets && (a->seq_capacity < 0 || (int64_t)a->num_seqs * a->seq_capacity > a->total_rows)) {
    return LA_ERROR_INVALID_VALUE;
  }
  if (a->num_seqs == 0) return LA_SUCCESS;
  if (!a->seq_lens || (a->total_rows > 0 && !a->kv_cache)) return LA_ERROR_INVALID_VALUE;
  if (a->tokens_per_seq > 0 && (!a->c_t || !a->k_rope)) return LA_ERROR_INVALID_VALUE;
  // per-sequence element counts stay within the kernel's 32-bit indexing
  if ((int64_t)a->tokens_per_seq * (a->cfg.kv_lora_rank + a->cfg.qk_rope_head_dim) > INT32_MAX ||
      (a->q_rope && (int64_t)a->queries_per_seq * a->cfg.num_heads * a->cfg.qk_rope_head_dim > INT32_MAX))
    return LA_ERROR_INVALID_VALUE;
  // the vectorised query rotation reads 16-B chunks of q_rope and the tables
  if (a->q_rope && (a->cfg.qk_rope_head_dim / 2) % 4 == 0 &&
      ((reinterpret_cast<uintptr_t>(a->q_rope) | reinterpret_cast<uintptr_t>(a->rope_cos) |
        reinterpret_cast<uintptr_t>(a->rope_sin)) & 15))
    return LA_ERROR_INVALID_VALUE;
  if (a->q_rope && (a->queries_per_seq < 1 || a->queries_per_seq > a->tokens_per_seq || !a->rope_cos ||
                    !a->rope_sin || (int64_t)a->num_seqs * a->queries_per_seq * a->cfg.num_heads > INT32_MAX))
    return LA_ERROR_INVALID_VALUE;
  la::AppendProblem p{};
  p.kv = a->kv_cache;
  p.kv_dtype = a->kv_dtype;
  p.total_rows = a->total_rows;
  p.num_seqs = a->num_seqs;
  p.capacity = a->seq_offsets ? 0 : a->seq_capacity;
  p.offsets = a->seq_offsets;
  p.lens = a->seq_lens;
  p.tokens = a->tokens_per_seq;
  p.c_t = a->c_t;
  p.k_rope = a->k_rope;
  p.src_dtype = a->src_dtype;
  p.q_rope = a->q_rope;
  p.qps = a->q_rope ? a->queries_per_seq : 0;
  p.nh = a->cfg.num_heads;
  p.rope_cos = a->rope_cos;
  p.rope_sin = a->rope_sin;
  p.rope_rows = a->rope_rows;
  p.status = a->status;
  p.dc = a->cfg.kv_lora_rank;
  p.dR = a->cfg.qk_rope_head_dim;
  if (paged) {
    p.block_table = a->block_table;
    p.block_size = a->block_size;
    p.blocks_per_seq = a->blocks_per_seq;
    p.pool_blocks = a->total_rows / a->block_size;
  }
  const hipError_t e = la::launch_append(p, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? (int)LA_SUCCESS : la::record_hip(e);
}

int la_absorb_q(const float* q_nope, const void* W_UK, int w_uk_dtype, float* q_absorbed, int tokens,
                const la_mla_config* cfg, void* stream) {
  if (!la::valid_cfg(cfg) || tokens < 0 || !la::valid_dtype(w_uk_dtype)) return LA_ERROR_INVALID_VALUE;
  if (tokens == 0) return LA_SUCCESS;
  if (!q_nope || !W_UK || !q_absorbed) return LA_ERROR_INVALID_VALUE;
  if (la::absorb_f32_supported(q_nope, W_UK, w_uk_dtype, q_absorbed, cfg->qk_nope_head_dim, cfg->kv_lora_rank)) {
    const hipError_t f = la::launch_absorb_f32(q_nope, W_UK, q_absorbed, tokens, cfg->num_heads, cfg->qk_nope_head_dim,
                                               cfg->kv_lora_rank, static_cast<hipStream_t>(stream));
    return f == hipSuccess ? (int)LA_SUCCESS : la::record_hip(f);
  }
  const bool mfma = la::absorb_mfma_supported(w_uk_dtype, cfg->num_heads, cfg->qk_nope_head_dim, cfg->kv_lora_rank) &&
                    (reinterpret_cast<uintptr_t>(q_nope) & 15) == 0 && (reinterpret_cast<uintptr_t>(W_UK) & 15) == 0;
  hipError_t e = mfma ? la::launch_absorb_mfma(q_nope, W_UK, w_uk_dtype, q_absorbed, 0, nullptr, 1.f, 0, tokens,
                                               cfg->num_heads, cfg->qk_nope_head_dim, cfg->kv_lora_rank, 1,
                                               static_cast<hipStream_t>(stream))
                      : la::launch_absorb(q_nope, W_UK, w_uk_dtype, q_absorbed, tokens, cfg->num_heads,
                                          cfg->qk_nope_head_dim, cfg->kv_lora_rank, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? (int)LA_SUCCESS : la::record_hip(e);
}

int la_mla_prefill(const la_prefill_args* args, void* stream) { return la::prefill(args, stream, true, nullptr); }

size_t la_mla_prefill_workspace_size(const la_prefill_args* args) {
  size_t need = 0;
  return la::prefill(args, nullptr, false, &need) == LA_SUCCESS ? need : 0;
}

int la_expand_prefix(const la_expand_args* args, void* stream) {
  return la::expand(args, static_cast<hipStream_t>(stream), true, nullptr);
}

size_t la_expand_prefix_workspace_size(const la_expand_args* args) {
  size_t need = 0;
  return la::expand(args, nullptr, false, &need) == LA_SUCCESS ? need : 0;
}

size_t la_expanded_size(int32_t rows, const la_mla_config* cfg) {
  if (!la::valid_cfg(cfg) || rows < 0 || !la::expanded_dims(*cfg)) return 0;
  const size_t tiles = ((size_t)rows + la::kTileKeys - 1) / la::kTileKeys;
  return tiles * (2 * (size_t)cfg->num_heads * la::kTileKBytes + la::kTileRBytes);
}

int la_mla_decode_shared(const la_shared_args* args, void* stream) {
  return la::decode_shared(args, static_cast<hipStream_t>(stream), true, nullptr);
}

size_t la_mla_decode_shared_workspace_size(const la_shared_args* args) {
  size_t need = 0;
  return la::decode_shared(args, nullptr, false, &need) == LA_SUCCESS ? need : 0;
}

}  // extern "C"
