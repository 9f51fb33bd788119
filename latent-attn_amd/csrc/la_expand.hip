// Latent rows -> per-head keys and values (the expanded form that prompts and
// shared prefixes attend over):
//   K[pos,h] = c_t[pos] . W_UK[h]^T   V[pos,h] = c_t[pos] . W_UV[h]^T   R[pos] = RoPE(k_rope[pos], pos)
// gather_kernel reads the cache once, whatever its layout and type, and
// writes 16-bit latent tiles of 64 rows (zeros past a sequence's last row, so
// nothing unfilled is ever an operand) and the rotated rope keys; the product
// then runs over dense rows, with sums in fp32 and one rounding to 16 bits, as
// the matrix instructions of the attention take them.
#include "la_prompt.hpp"

#include <type_traits>

namespace la {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lchar;

template <typename T>
struct Mm;
template <>
struct Mm<__hip_bfloat16> {
  typedef bf16x8 vec;
  typedef __bf16 elem;
  static __device__ inline f32x16 mma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mm<__half> {
  typedef f16x8 vec;
  typedef _Float16 elem;
  static __device__ inline f32x16 mma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// Values past fp16's range. A weight of zero times infinity is NaN, so an
// infinite value would reach the tokens that do not see its row. It becomes the
// largest number, and over(row of the block) is called by a lane that holds one,
// for a NaN in the row's key: that reaches the tokens that see it, through their
// scores. (bf16 has fp32's range, whose end no other form passes either.)
constexpr float kHalfMost = 65504.f, kHalfOver = 65520.f;  // from kHalfOver on fp16 rounds to infinity
template <int kBlocks>
__device__ inline bool past_half(const f32x16 (&v)[kBlocks]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kBlocks; ++i)
#pragma unroll
    for (int e = 0; e < 16; e += 2)
      asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(top) : "v"(top), "v"(v[i][e]), "v"(v[i][e + 1]));
  return __builtin_amdgcn_ballot_w64(top >= kHalfOver) != 0;
}
template <typename Over>
__device__ inline void hold_half(f32x16& v, int g, Over over) {  // a block of 32 rows: 8 (e / 4) + 4 g + e % 4 in register e
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (fabsf(v[e]) >= kHalfOver) {
      v[e] = copysignf(kHalfMost, v[e]);
      over(8 * (e >> 2) + 4 * g + (e & 3));
    }
}

// ---- gather --------------------------------------------------------------------

// Eight cache elements as T (an 8-bit cache: bf16, exact).
template <typename KT, typename T, bool kAligned>
__device__ inline typename Mm<T>::vec load8(const KT* p) {
  typedef typename Mm<T>::vec vec;
  KT b[8];
  if constexpr (kAligned) __builtin_memcpy(b, __builtin_assume_aligned(p, 8 * sizeof(KT)), sizeof(b));
  else __builtin_memcpy(b, p, sizeof(b));
  if constexpr (sizeof(KT) == 2) {
    return __builtin_bit_cast(vec, b);
  } else {
    uint32_t w[2], y[4];
    __builtin_memcpy(w, b, 8);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      y[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.f, false));
      y[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.f, true));
    }
    return __builtin_bit_cast(vec, y);
  }
}

// kGatherRows rows of a tile per workgroup, a row per wave at a time; the
// workgroups behind the tiles find the query tiles. A row whose latent holds an
// infinity or NaN gets zeros there and NaN as its rope key: the tokens that see
// it get NaN through their scores, as from its values, and those that do not
// (their weight is zero, and zero times NaN is NaN) are left alone. Bound by
// memory's latency and then its bytes: 8192 rows 9 us (18 MB), 23,800 8-bit rows
// 13 us.
constexpr int kGatherRows = 16;
constexpr int kGatherParts = kTileKeys / kGatherRows;
// Sequence of a tile, the position of its first row and its rows.
struct TileRows {
  int s, pos0, rows;
};
__device__ inline TileRows tile_rows_of(const RowSource& src, int64_t tile) {
  const int s = source_find(src, tile);
  const int64_t t = tile - source_tile(src, s);  // < 0: rows before the first sequence
  const int L = t < 0 ? 0 : source_rows(src, s);
  return TileRows{s, (int)t * kTileKeys, (int)clamp64(L - t * kTileKeys, 0, L > 0 ? kTileKeys : 0)};
}
// Rows r0 + step i (i < kN) of a tile by one wave, eight elements per lane, to
// put(row, elements); bit i of the result: row i was not finite.
template <typename KT, typename T, bool kAligned, int kN, typename Put>
__device__ inline uint32_t latent_rows(const RowSource& src, const TileRows& tr, int r0, int step, int lane, Put put) {
  typedef typename Mm<T>::vec vec;
  const KT* const kv = static_cast<const KT*>(src.kv);
  vec v[kN] = {};
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int r = r0 + step * i;
    if (r < tr.rows) v[i] = load8<KT, T, kAligned>(kv + source_row(src, tr.s, tr.pos0 + r) * src.row_elems + 8 * lane);
  }
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    float z = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) z = __builtin_fmaf((float)v[i][e], 0.f, z);
    if (__builtin_amdgcn_ballot_w64(!(z == 0.f)) != 0) {
      v[i] = vec{};
      bad |= 1u << i;
    }
    put(r0 + step * i, v[i]);
  }
  return bad;
}
// Piece `block` of the gather by 4 waves: kGatherRows rows of a tile, or 256 query
// tiles. kRows: the latent rows and the tile's row count are stored, not the rope keys alone.
template <typename KT, typename T, bool kAligned, bool kRows>
__device__ inline void gather_piece(const ExpandProblem& p, int64_t block, int wave, int lane) {
  typedef typename Mm<T>::vec vec;
  typedef typename Mm<T>::elem elem;
  typedef elem vec4 __attribute__((ext_vector_type(4)));
  const int64_t tile = block / kGatherParts;
  if (tile >= p.src.num_tiles) {
    const int64_t qt = (block - p.src.num_tiles * kGatherParts) * 256 + 64 * wave + lane;
    if (qt < p.q_tiles) p.q_info[qt] = make_query_tile(p.q, p.src, qt, p.query_rows);
    return;
  }
  const TileRows tr = tile_rows_of(p.src, tile);
  const int r0 = (int)(block % kGatherParts) * kGatherRows + wave;
  if (kRows && r0 == 0 && lane == 0) p.tile_rows[tile] = tr.rows;
  if (tr.rows == 0) return;
  // the wave's rope keys, 8 lanes a row: dims d .. d + 3 and their partners d + 32 ..
  const int r = r0 + 4 * (lane >> 3 & 3), d = 4 * (lane & 7);
  float k0[4] = {}, k1[4] = {}, c[4] = {}, sn[4] = {};
  if (r < tr.rows) {
    const KT* const k = static_cast<const KT*>(p.src.kv) + source_row(p.src, tr.s, tr.pos0 + r) * p.src.row_elems + 512 + d;
    const int64_t at = source_rope_row(p.src, tr.pos0 + r) * 32 + d;
    KT b0[4], b1[4];
    if constexpr (kAligned) {
      __builtin_memcpy(b0, __builtin_assume_aligned(k, sizeof(b0)), sizeof(b0));
      __builtin_memcpy(b1, __builtin_assume_aligned(k + 32, sizeof(b1)), sizeof(b1));
    } else {
      __builtin_memcpy(b0, k, sizeof(b0));
      __builtin_memcpy(b1, k + 32, sizeof(b1));
    }
    __builtin_memcpy(c, p.src.cos + at, sizeof(c));
    __builtin_memcpy(sn, p.src.sin + at, sizeof(sn));
#pragma unroll
    for (int e = 0; e < 4; ++e) k0[e] = to_f32(b0[e]), k1[e] = to_f32(b1[e]);
  }
  vec* const c_out = reinterpret_cast<vec*>(static_cast<char*>(p.rows_c) + tile * kTileCBytes);
  const uint32_t bad = latent_rows<KT, T, kAligned, kGatherRows / 4>(p.src, tr, r0, 4, lane, [&](int row, const vec& v) {
    if constexpr (kRows) c_out[row * 64 + lane] = v;
  });
  if (lane >= 32) return;
  vec4 a, b;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    a[e] = (elem)((k0[e] * c[e] - k1[e] * sn[e]) * p.k_scale);
    b[e] = (elem)((k0[e] * sn[e] + k1[e] * c[e]) * p.k_scale);
  }
  const elem nan = (elem)__builtin_nanf("");
  if (bad >> (lane >> 3) & 1) a = b = vec4{nan, nan, nan, nan};
  elem* const r_out = reinterpret_cast<elem*>(static_cast<char*>(p.rope) + tile * kTileRBytes);
  elem* const o = r_out + (r >> 5) * (4 * 512) + operand_elem(r, d & 15);
  *reinterpret_cast<vec4*>(o + (d >> 4) * 512) = a;
  *reinterpret_cast<vec4*>(o + ((d >> 4) + 2) * 512) = b;
}
template <typename KT, typename T, bool kAligned>
__global__ __launch_bounds__(256) void gather_kernel(ExpandProblem p) {
  gather_piece<KT, T, kAligned, true>(p, blockIdx.x, __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), threadIdx.x & 63);
}

__global__ __launch_bounds__(256) void convert_kernel(const void* src, int src_dtype, uint16_t* dst, int f16, int64_t n) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step) {
    const float x = load_any(src, src_dtype, i);
    dst[i] = f16 ? __builtin_bit_cast(uint16_t, (_Float16)x) : __builtin_bit_cast(uint16_t, (__bf16)x);
  }
}

// ---- expand ----------------------------------------------------------------------

// One head's 256 weight rows (128 of W_UK, then 128 of W_UV) times 64 kPb
// positions per workgroup of 8 waves: a quarter of the weight rows (0, 1: K
// dims; 2, 3: V dims) by half of the positions each. Stages of kBk latent
// columns in a ring in LDS: one is read, the others are on their way. 16-byte
// chunk j of row r lies at j ^ (r / 2 % 8), which the copies' addresses apply:
// rows are half as long as all banks, so 16 rows' chunks fill them.
//
// The rows and weights that pass the L2 bound it, not its products (with the
// copies left out 8192 rows x 128 heads took 234 us for 334, with the products
// left out 301): hence the large tile, and the order in which an XCD takes its
// items. Large calls run a workgroup per CU, which takes items in turn and has
// the next one's first stage on its way while it stores (4 tiles); small ones
// a workgroup per item and tile, with three stages on their way. 8192 rows x
// 128 heads: 275 GFLOP in 275 us, 1.0 PFLOP/s (a library product of the shape,
// which writes them in no such order, 371); 1001 rows 36 us (when it was chosen 39,
// of 47 in workgroups of one tile and 51 in two of them per CU).
constexpr int kDc = 512;
constexpr int kBk = 64;
constexpr int kStages = kDc / kBk;
constexpr int kRowBytes = kBk * 2;
constexpr int kNRows = 256;
template <int kPb>
struct Geometry {  // kPb tiles per item, blocks of 32 positions per wave
  static constexpr int kPos = 64 * kPb;
  static constexpr int kRing = kPb == 4 ? 2 : 4;
  static constexpr int kStageBytes = (kPos + kNRows) * kRowBytes;
  static constexpr int kCopies = kStageBytes / 1024 / 8;  // of 1 KB (8 rows) per wave and stage
  static constexpr int kStores = 4 * kPb;                  // of a wave and item
  static_assert(kCopies * 8 * 8 == kPos + kNRows, "every row of a stage is copied once");
};
// Heads that an XCD takes together: their weights (1 MB) stay in its L2 while
// all rows pass, once per group (all 16 heads of an XCD per block of rows: more
// weights than an L2 holds, again for every block).
__host__ __device__ inline int head_group(int heads) { return heads > 24 ? 4 : (heads + 7) / 8; }
__host__ __device__ inline int64_t items_per_xcd(int heads, int64_t tiles, int pb) {
  const int group = head_group(heads);
  return (int64_t)((heads + 8 * group - 1) / (8 * group) * group) * ((tiles + pb - 1) / pb);
}

template <int N>
__device__ inline void wait_copies() {
  static_assert(N == 0 || N == 4 || N == 10 || N == 16, "");
  if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  else if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  else if constexpr (N == 10) asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
}

// The work of one wave (kV: of V dims). Both kinds have the same barriers; each
// has its own accumulators, since a branch around the products alone made the
// compiler copy and spill them.
template <typename T, int kPb, bool kV>
__device__ inline void expand_wave(const ExpandProblem& p, int64_t step, lchar* L, int lane, int wave) {
  typedef typename Mm<T>::vec vec;
  typedef typename Mm<T>::elem elem;
  typedef const __attribute__((address_space(3))) vec lvec;
  typedef Geometry<kPb> G;
  // Items of an XCD (id % 8), every step-th from id / 8 on: head of the group
  // fastest, then rows, then groups; heads past the last and empty tiles are no items.
  const int64_t blocks = (p.src.num_tiles + kPb - 1) / kPb, items = items_per_xcd(p.heads, p.src.num_tiles, kPb);
  const int group = head_group(p.heads);
  int64_t item = blockIdx.x >> 3, tile0 = 0;
  int h = 0;
  auto find = [&]() {  // the first item from `item` on, or items
    for (; item < items; item += step) {
      h = (int)(blockIdx.x & 7) + 8 * ((int)(item / group / blocks) * group + (int)(item % group));
      tile0 = item / group % blocks * kPb;
      int any = 0;
#pragma unroll
      for (int i = 0; i < kPb; ++i) any |= tile0 + i < p.src.num_tiles ? p.tile_rows[tile0 + i] : 0;
      if (h < p.heads && any != 0) return;
    }
  };
  const char* base[G::kCopies];
  uint32_t off[G::kCopies];
  auto sources = [&] {
    // rows past the last tile (whose products nobody stores) read the last row
    const int rows = (int)clamp64((p.src.num_tiles - tile0) * kTileKeys, 0, G::kPos);
    const char* const X = static_cast<const char*>(p.rows_c) + tile0 * kTileCBytes;
    const char* const WK = static_cast<const char*>(p.W_UK) + (int64_t)(p.head0 + h) * 128 * kDc * 2;
    const char* const WV = static_cast<const char*>(p.W_UV) + (int64_t)(p.head0 + h) * 128 * kDc * 2;
    const int r = lane >> 3;
#pragma unroll
    for (int i = 0; i < G::kCopies; ++i) {
      const int r0 = 8 * (G::kCopies * wave + i);  // a copy's rows are all X's, W_UK's or W_UV's
      base[i] = r0 < G::kPos ? X : r0 < G::kPos + 128 ? WK + (r0 - G::kPos) * (kDc * 2) : WV + (r0 - G::kPos - 128) * (kDc * 2);
      off[i] = (uint32_t)((r0 < G::kPos ? min(r0 + r, rows - 1) : r) * (kDc * 2) +
                          16 * ((lane & 7) ^ (4 * ((G::kCopies * wave + i) & 1) + (r >> 1))));
    }
  };
  // inline asm without outputs: behind the builtin the compiler waits for every LDS read at once
  auto issue = [&](int k) {
    const uint32_t buf = (uint32_t)(uintptr_t)L + k % G::kRing * G::kStageBytes + 1024 * G::kCopies * wave;
    const int kk = min(k, kStages - 1);  // past the end (small calls): the last stage again, never read
#pragma unroll
    for (int i = 0; i < G::kCopies; ++i)
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(buf + 1024 * i), "v"(off[i]),
                   "s"(base[i] + kk * kRowBytes)
                   : "memory", "m0");
  };
  const int wn = wave & 3, wp = wave >> 2;  // weight quarter, position half
  const int r32 = lane & 31, g = lane >> 5;
  const lchar* const wr = L + (G::kPos + 64 * wn + r32) * kRowBytes;
  const lchar* const xr = L + (32 * kPb * wp + r32) * kRowBytes;
  find();
  if (item >= items) return;
  sources();
#pragma unroll
  for (int k = 0; k < G::kRing - 1; ++k) issue(k);
  bool stored = false;  // the copies on their way are behind kStores stores
  while (true) {
    f32x16 acc[kPb][2] = {};
    vec w[2][2], x[2][kPb];
    const int64_t out_tile = tile0;
    const int out_h = h;
    bool more = false;
#pragma unroll 1
    for (int k = 0; k < kStages; ++k) {
      // this wave's copies of stage k have landed; everyone's, and stage k - 1 is read
      if (kPb == 4 && k == 0 && stored) wait_copies<G::kRing == 2 ? 16 : 0>();
      else wait_copies<(G::kRing - 2) * G::kCopies>();
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (kPb == 4 && k == kStages - 1) {
        item += step;
        find();
        more = item < items;
        if (more) {
          sources();
          issue(0);
        }
      } else {
        issue(k + G::kRing - 1);
      }
      const int at = k % G::kRing * G::kStageBytes;
      auto read = [&](int ks) {
        const int c = at + 16 * ((2 * ks + g) ^ (r32 >> 1 & 7));
#pragma unroll
        for (int j = 0; j < 2; ++j) w[ks & 1][j] = *reinterpret_cast<lvec*>(wr + 32 * j * kRowBytes + c);
#pragma unroll
        for (int i = 0; i < kPb; ++i) x[ks & 1][i] = *reinterpret_cast<lvec*>(xr + 32 * i * kRowBytes + c);
      };
      read(0);
#pragma unroll
      for (int ks = 0; ks < kBk / 16; ++ks) {
        if (ks + 1 < kBk / 16) read(ks + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kPb; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            acc[i][j] = kV ? Mm<T>::mma(x[ks & 1][i], w[ks & 1][j], acc[i][j]) : Mm<T>::mma(w[ks & 1][j], x[ks & 1][i], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int i = 0; i < kPb; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) settle(acc[i][j]);
    if constexpr (kV && std::is_same<T, __half>::value) {
#pragma unroll
      for (int i = 0; i < kPb; ++i) {
        const int pb = kPb * wp + i;
        const int64_t tile = out_tile + pb / 2;
        if (tile < p.src.num_tiles && past_half(acc[i])) {
          _Float16* const rope = static_cast<_Float16*>(p.rope) + tile * (kTileRBytes / 2) + (pb & 1) * (4 * 512);
#pragma unroll
          for (int j = 0; j < 2; ++j)
            hold_half(acc[i][j], g, [&](int row) { rope[operand_elem(row, 0)] = (_Float16)__builtin_nanf(""); });
        }
      }
    }
    // registers 8 q .. 8 q + 7 of a block are one operand element group (operand
    // order, la_prompt.hpp): K: a step of 16 dims; V: of 16 keys
#pragma unroll
    for (int i = 0; i < kPb; ++i) {
      const int pb = kPb * wp + i;  // block of 32 positions
      const int64_t tile = out_tile + pb / 2;
      if (tile >= p.src.num_tiles) continue;
      char* const out = static_cast<char*>(kV ? p.vx : p.kx) + ((int64_t)out_h * p.src.num_tiles + tile) * kTileKBytes;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          vec v;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = (elem)(kV ? acc[i][j][8 * q + e] : acc[i][j][8 * q + e] * p.k_scale);
          const int db = 2 * (wn & 1) + j;  // block of 32 dims
          const int piece = kV ? 4 * db + 2 * (pb & 1) + q : 8 * (pb & 1) + 2 * db + q;
          *reinterpret_cast<vec*>(out + piece * 1024 + 16 * lane) = v;
        }
    }
    if (kPb != 4 || !more) break;
    stored = out_tile + kPb <= p.src.num_tiles;  // all of them: else the next wait takes everything
  }
  wait_copies<0>();  // the copies past the end have landed: the workgroup may end
}

template <typename T, int kPb>
__global__ __launch_bounds__(512, 2) void expand_kernel(ExpandProblem p, int64_t step) {
  extern __shared__ __attribute__((aligned(1024))) char expand_lds[];
  lchar* const L = (lchar*)expand_lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if ((wave & 3) >= 2) expand_wave<T, kPb, true>(p, step, L, lane, wave);
  else expand_wave<T, kPb, false>(p, step, L, lane, wave);
}

template <typename T, int kPb>
hipError_t expand_pb(const ExpandProblem& p, hipStream_t stream, int ncu) {
  constexpr int lds = Geometry<kPb>::kRing * Geometry<kPb>::kStageBytes;
  static OncePerDevice once;
  hipError_t e = allow_lds(once, reinterpret_cast<const void*>(expand_kernel<T, kPb>), lds);
  if (e != hipSuccess) return e;
  int64_t per_xcd = items_per_xcd(p.heads, p.src.num_tiles, kPb);
  if (kPb == 4) per_xcd = per_xcd < (ncu + 7) / 8 ? per_xcd : (ncu + 7) / 8;
  if (8 * per_xcd > most_blocks(512)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((expand_kernel<T, kPb>), dim3((unsigned)(8 * per_xcd)), dim3(512), lds, stream, p, per_xcd);
  return hipGetLastError();
}

// ---- gather and expand in one: small calls ---------------------------------------------

// A workgroup of 8 waves per (head, tile): its 64 latent rows to LDS, then the
// product as in expand_kernel, the weights in a ring of three stages whose
// copies are on their way before the rows are looked up. The workgroups behind
// the items write the rope keys and query tiles, two pieces of the gather each.
// Latency of its loads: 17 rows x 16 heads 8 us (gather and expansion one after
// the other 12), 300 x 16 a call 9.3 (11.2).
constexpr int kSmallW = kNRows * kRowBytes;  // a stage of weights
constexpr int kSmallRing = 3;
constexpr int kSmallX = kTileKeys * kDc * 2;
constexpr int kSmallLds = kSmallX + kSmallRing * kSmallW;
static_assert(kSmallLds <= 160 * 1024, "LDS of a CU");

// Stage k of the weights into its part of the ring: four copies of 8 rows per
// wave (32 rows from W on); past the end the last stage again, never read.
__device__ inline void small_issue(lchar* L, const char* W, uint32_t off, int k, int wave) {
  const uint32_t buf = (uint32_t)(uintptr_t)L + kSmallX + k % kSmallRing * kSmallW + 4096 * wave;
  const char* const from = W + min(k, kStages - 1) * kRowBytes;
#pragma unroll
  for (int i = 0; i < 4; ++i)  // (odd groups of 8 rows: 4 in the swizzle's row pairs)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(buf + 1024 * i),
                 "v"(off ^ (i & 1 ? 64u : 0u)), "s"(from + i * 8 * (kDc * 2))
                 : "memory", "m0");
}
template <typename T, bool kV>
__device__ inline void small_products(const ExpandProblem& p, lchar* L, int64_t tile, int h, int lane, int wave,
                                      const char* W, uint32_t off) {
  typedef typename Mm<T>::vec vec;
  typedef typename Mm<T>::elem elem;
  typedef const __attribute__((address_space(3))) vec lvec;
  const int wn = wave & 3, wp = wave >> 2, r32 = lane & 31, g = lane >> 5;
  f32x16 acc[2] = {};
  const lchar* const xr = L + (32 * wp + r32) * (kDc * 2);
  const lchar* const wr = L + kSmallX + (64 * wn + r32) * kRowBytes;
#pragma unroll 1
  for (int k = 0; k < kStages; ++k) {
    wait_copies<4>();  // this wave's of stage k have landed, those of the next may be on their way
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    small_issue(L, W, off, k + kSmallRing - 1, wave);
    const lchar* const w0 = wr + k % kSmallRing * kSmallW;
#pragma unroll
    for (int ks = 0; ks < kBk / 16; ++ks) {
      vec w[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        w[j] = *reinterpret_cast<lvec*>(w0 + 32 * j * kRowBytes + 16 * ((2 * ks + g) ^ (r32 >> 1 & 7)));
      const vec x = *reinterpret_cast<lvec*>(xr + 16 * ((8 * k + 2 * ks + g) ^ (r32 & 15)));
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[j] = kV ? Mm<T>::mma(x, w[j], acc[j]) : Mm<T>::mma(w[j], x, acc[j]);
    }
  }
  const int64_t at = ((int64_t)h * p.src.num_tiles + tile) * kTileKBytes;
  char* const out = static_cast<char*>(kV ? p.vx : p.kx) + at;
#pragma unroll
  for (int j = 0; j < 2; ++j) settle(acc[j]);
  uint32_t over = 0;  // fp16: this lane's rows of the block with a value past the range
  if constexpr (kV && std::is_same<T, __half>::value) {
    if (past_half(acc))
#pragma unroll
      for (int j = 0; j < 2; ++j) hold_half(acc[j], g, [&](int row) { over |= 1u << row; });
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      vec v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (elem)(kV ? acc[j][8 * q + e] : acc[j][8 * q + e] * p.k_scale);
      const int db = 2 * (wn & 1) + j;  // block of 32 dims
      const int piece = kV ? 4 * db + 2 * wp + q : 8 * wp + 2 * db + q;
      *reinterpret_cast<vec*>(out + piece * 1024 + 16 * lane) = v;
    }
  }
  if constexpr (std::is_same<T, __half>::value) {
    // the rope keys are other workgroups', so a NaN goes into this head's key, behind the stores of the keys
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    _Float16* const key = reinterpret_cast<_Float16*>(static_cast<char*>(p.kx) + at) + wp * (8 * 512);
    for (; over; over &= over - 1) key[operand_elem(__builtin_ctz(over), 0)] = (_Float16)__builtin_nanf("");
  }
}

template <typename KT, typename T, bool kAligned>
__global__ __launch_bounds__(512, 2) void gather_expand_kernel(ExpandProblem p, int64_t items) {
  extern __shared__ __attribute__((aligned(1024))) char small_lds[];
  typedef typename Mm<T>::vec vec;
  lchar* const L = (lchar*)small_lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (blockIdx.x >= items) {
    const int64_t pieces = p.src.num_tiles * kGatherParts + (p.q_tiles + 255) / 256;
    const int64_t piece = 2 * ((int64_t)blockIdx.x - items) + (wave >> 2);
    if (piece < pieces) gather_piece<KT, T, kAligned, false>(p, piece, wave & 3, lane);
    return;
  }
  const int per = (p.heads + 7) / 8, k = blockIdx.x >> 3, h = k % per * 8 + (blockIdx.x & 7);  // a head's on one XCD
  const int64_t tile = k / per;
  if (h >= p.heads) return;
  // Copies of a stage: 4 of a wave's, 8 weight rows of 128 B each; its rows are all W_UK's or W_UV's.
  const char* const W = static_cast<const char*>(wave < 4 ? p.W_UK : p.W_UV) +
                        ((int64_t)(p.head0 + h) * 128 + 32 * (wave & 3)) * (kDc * 2);
  const int r = lane >> 3;
  const uint32_t off = (uint32_t)(r * (kDc * 2)) + 16 * ((lane & 7) ^ (r >> 1));  // of an even group of 8 rows
#pragma unroll
  for (int i = 0; i < kSmallRing - 1; ++i) small_issue(L, W, off, i, wave);
  const TileRows tr = tile_rows_of(p.src, tile);
  if (tr.rows > 0) {
    latent_rows<KT, T, kAligned, 8>(p.src, tr, wave, 8, lane, [&](int row, const vec& v) {
      typedef __attribute__((address_space(3))) vec lvec;
      *reinterpret_cast<lvec*>(L + row * (kDc * 2) + 16 * (lane ^ (row & 15))) = v;
    });
    if ((wave & 3) >= 2) small_products<T, true>(p, L, tile, h, lane, wave, W, off);
    else small_products<T, false>(p, L, tile, h, lane, wave, W, off);
  }
  wait_copies<0>();  // all copies have landed: the workgroup may end
}

template <typename KT, typename T>
hipError_t gather_expand_t(const ExpandProblem& p, bool aligned, hipStream_t stream) {
  const void* const k = aligned ? reinterpret_cast<const void*>(gather_expand_kernel<KT, T, true>)
                                : reinterpret_cast<const void*>(gather_expand_kernel<KT, T, false>);
  static OncePerDevice once[2];
  const hipError_t e = allow_lds(once[aligned], k, kSmallLds);
  if (e != hipSuccess) return e;
  const int64_t items = 8 * (int64_t)((p.heads + 7) / 8) * p.src.num_tiles;
  const int64_t pieces = p.src.num_tiles * kGatherParts + (p.q_tiles + 255) / 256;
  const int64_t blocks = items + (pieces + 1) / 2;
  if (blocks > most_blocks(512)) return hipErrorInvalidValue;
  if (aligned)
    hipLaunchKernelGGL((gather_expand_kernel<KT, T, true>), dim3((unsigned)blocks), dim3(512), kSmallLds, stream, p, items);
  else
    hipLaunchKernelGGL((gather_expand_kernel<KT, T, false>), dim3((unsigned)blocks), dim3(512), kSmallLds, stream, p, items);
  return hipGetLastError();
}

int64_t gather_blocks(int64_t tiles, int64_t q_tiles) { return tiles * kGatherParts + (q_tiles + 255) / 256; }

template <typename KT, typename T>
hipError_t gather_t(const ExpandProblem& p, bool aligned, hipStream_t stream) {
  const dim3 grid((unsigned)gather_blocks(p.src.num_tiles, p.q_tiles));
  if (aligned) hipLaunchKernelGGL((gather_kernel<KT, T, true>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((gather_kernel<KT, T, false>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

// Gathers in the expansion's workgroups, one per (head, tile), where half the
// CUs hold them (us a call, three launches / two: 17 tokens x 16 heads 20.4 /
// 17.4, x 128 22.8 / 18.5, 256 x 16 29.6 / 27.5; one per CU, 1000 x 16 43.9 / 45.0;
// two per CU, 250 x 128 38.4 / 44.4: every head reads and converts the rows).
bool small_call(const ExpandProblem& p, int ncu) {
  return p.src.num_tiles > 0 && 2 * (int64_t)p.heads * p.src.num_tiles <= ncu;
}

}  // namespace

bool expand_fits(int64_t tiles, int64_t q_tiles) { return gather_blocks(tiles, q_tiles) <= most_blocks(256); }

hipError_t launch_gather(const ExpandProblem& p, hipStream_t stream, int ncu) {
  if (small_call(p, ncu) || (p.src.num_tiles == 0 && p.q_tiles == 0)) return hipSuccess;
  if (!expand_fits(p.src.num_tiles, p.q_tiles) || p.src.row_elems != 576) return hipErrorInvalidValue;
  const bool aligned = (reinterpret_cast<uintptr_t>(p.src.kv) & 15) == 0;  // rows are 1152 or 576 B
  switch (p.src.kv_dtype) {
    case LA_DTYPE_BF16: return gather_t<__hip_bfloat16, __hip_bfloat16>(p, aligned, stream);
    case LA_DTYPE_F16: return gather_t<__half, __half>(p, aligned, stream);
    case LA_DTYPE_FP8_E4M3: return gather_t<fp8e4m3, __hip_bfloat16>(p, aligned, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_expand(const ExpandProblem& p, hipStream_t stream, int ncu) {
  if (p.src.num_tiles == 0 || p.heads == 0) return hipSuccess;
  if (small_call(p, ncu)) {
    if (!expand_fits(p.src.num_tiles, p.q_tiles) || p.src.row_elems != 576) return hipErrorInvalidValue;
    const bool aligned = (reinterpret_cast<uintptr_t>(p.src.kv) & 15) == 0;
    switch (p.src.kv_dtype) {
      case LA_DTYPE_BF16: return gather_expand_t<__hip_bfloat16, __hip_bfloat16>(p, aligned, stream);
      case LA_DTYPE_F16: return gather_expand_t<__half, __half>(p, aligned, stream);
      case LA_DTYPE_FP8_E4M3: return gather_expand_t<fp8e4m3, __hip_bfloat16>(p, aligned, stream);
      default: return hipErrorInvalidValue;
    }
  }
  const bool wide = (int64_t)p.heads * ((p.src.num_tiles + 3) / 4) >= ncu;
  if (p.f16) return wide ? expand_pb<__half, 4>(p, stream, ncu) : expand_pb<__half, 1>(p, stream, ncu);
  return wide ? expand_pb<__hip_bfloat16, 4>(p, stream, ncu) : expand_pb<__hip_bfloat16, 1>(p, stream, ncu);
}

hipError_t launch_convert(const void* src, int src_dtype, void* dst, int f16, int64_t n, hipStream_t stream) {
  if (n == 0) return hipSuccess;
  const int64_t blocks = n / 1024 + 1 < 4096 ? n / 1024 + 1 : 4096;
  hipLaunchKernelGGL(convert_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, src, src_dtype,
                     static_cast<uint16_t*>(dst), f16, n);
  return hipGetLastError();
}

}  // namespace la
