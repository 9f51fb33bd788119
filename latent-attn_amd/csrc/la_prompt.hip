// Attention of many tokens per sequence over expanded keys and values
// (la_mla_prefill; the prefix part of la_mla_decode_shared), and the kernels
// around it: the plain form for other types and head shapes, and the queries
// of the absorbed form.
//
//   s[q,k] = scale * (q_nope[q] . K[k] + q_rope[q] . R[k]),  k < visible(q)
//   out[q] = softmax_k(s[q]) . V
// in one pass over the keys with a running maximum m and sum l per query.
#include "la_prompt.hpp"

namespace la {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
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

constexpr int kQRows = 32;              // queries per wave
constexpr int kQBlock = 4 * kQRows;     // and per workgroup
constexpr int kBufBytes = 2 * kTileKBytes + kTileRBytes;  // K, V, rope keys of one tile
constexpr float kSlack = 8.f;           // the running maximum rises by more than this or stays
constexpr float kNoScore = -1e30f;      // below every score: the maximum before the first one

// Four wait states more than an accumulator needs before its first VALU reader
// (the compiler adds none where a branch lies between).
template <typename V>
__device__ inline void settle2(V& a, V& b) { asm volatile("s_nop 15\n\ts_nop 7" : "+v"(a), "+v"(b)); }

__device__ inline void store1(void* out, int dtype, int64_t i, float v) {
  if (dtype == LA_DTYPE_F32) static_cast<float*>(out)[i] = v;
  else if (dtype == LA_DTYPE_BF16) static_cast<__bf16*>(out)[i] = (__bf16)v;
  else static_cast<_Float16*>(out)[i] = (_Float16)v;
}

// The query of one lane as operands: 12 steps of 8 elements, step by step {16 k +
// 4 g + (0..3), 16 k + 8 + 4 g + (0..3)}. All loads go out before the first is
// waited for, so the type decides around them, not between them. Queries and
// outputs are a good part of a short prompt (512 tokens x 128 heads: 18 us beside
// 2.2 per tile of keys), in 16 B per lane where they allow it (16 x 300 tokens,
// a call: 408 us in pieces of 8 B, 398 with such loads, 384 with such stores
// too; 1001 tokens 102, 98, 97; 17 x 16 heads 17.4, 17.3, 16.6).
enum QueryLoad { kScalar, kVec16, kVec32, kWide16 };
template <typename T, QueryLoad kLoad>
__device__ inline void load_query_as(const PromptProblem& p, int64_t an, int64_t ar, int64_t pos, int g,
                                     typename Mm<T>::vec (&qn)[8], typename Mm<T>::vec (&qr)[4]) {
  typedef typename Mm<T>::elem elem;
  float x[24][4];  // 16 pieces of the nope part, 8 of the rope part
  auto at = [&](int i) { return i < 16 ? an + 8 * i + 4 * g : ar + 8 * (i - 16) + 4 * g; };
  if constexpr (kLoad == kVec16 || kLoad == kWide16) {
    uint2 w[24];
    if constexpr (kLoad == kVec16) {
#pragma unroll
      for (int i = 0; i < 24; ++i)
        w[i] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(i < 16 ? p.q.q_nope : p.q.q_rope) + at(i));
    } else {  // 16 B per lane, the halves' middle pieces exchanged
      uint4 v[12];
#pragma unroll
      for (int i = 0; i < 12; ++i)
        v[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(i < 8 ? p.q.q_nope : p.q.q_rope) +
                                               (i < 8 ? an + 16 * i : ar + 16 * (i - 8)) + 8 * g);
#pragma unroll
      for (int i = 0; i < 12; ++i) {
        const auto x = __builtin_amdgcn_permlane32_swap(v[i].x, v[i].z, false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(v[i].y, v[i].w, false, false);
        w[2 * i] = uint2{x[0], y[0]};
        w[2 * i + 1] = uint2{x[1], y[1]};
      }
    }
    const bool bf16 = p.q.dtype == LA_DTYPE_BF16;
#pragma unroll
    for (int i = 0; i < 24; ++i) {
      const uint32_t b[4] = {w[i].x & 0xFFFF, w[i].x >> 16, w[i].y & 0xFFFF, w[i].y >> 16};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[i][e] = bf16 ? f_of(b[e] << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)b[e]);
    }
  } else if constexpr (kLoad == kVec32) {
#pragma unroll
    for (int i = 0; i < 24; ++i) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(static_cast<const float*>(i < 16 ? p.q.q_nope : p.q.q_rope) + at(i));
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = v[e];
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < 24; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = load_any(i < 16 ? p.q.q_nope : p.q.q_rope, p.q.dtype, at(i) + e);
#pragma unroll
        for (int k = 0; k < 24; ++k) x[k][e] = k == i ? v : x[k][e];
      }
  }
  if (p.q.rotate) {
    f32x4 c[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* const cp = p.src.cos + pos + 8 * i + 4 * g;
      const float* const sp = p.src.sin + pos + 8 * i + 4 * g;
      if (p.table_vec) {
        c[i] = *reinterpret_cast<const f32x4*>(cp);
        s[i] = *reinterpret_cast<const f32x4*>(sp);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) c[i][e] = cp[e], s[i][e] = sp[e];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = x[16 + i][e], b = x[20 + i][e];
        x[16 + i][e] = a * c[i][e] - b * s[i][e];
        x[20 + i][e] = a * s[i][e] + b * c[i][e];
      }
  }
#pragma unroll
  for (int i = 0; i < 24; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i < 16) qn[i >> 1][4 * (i & 1) + e] = (elem)(x[i][e] * p.q_scale);
      else qr[(i - 16) >> 1][4 * (i & 1) + e] = (elem)(x[i][e] * p.q_scale);
    }
}
template <typename T>
__device__ inline void load_query(const PromptProblem& p, int64_t token, int h, int64_t pos, int g,
                                  typename Mm<T>::vec (&qn)[8], typename Mm<T>::vec (&qr)[4]) {
  const int64_t an = token * p.q.nope_stride + h * p.q.nope_head, ar = token * p.q.rope_stride + h * p.q.rope_head;
  const int64_t at = source_rope_row(p.src, pos) * 32;
  if (!(p.nope_vec && p.rope_vec)) load_query_as<T, kScalar>(p, an, ar, at, g, qn, qr);
  else if (p.q.dtype == LA_DTYPE_F32) load_query_as<T, kVec32>(p, an, ar, at, g, qn, qr);
  else if (p.q_wide) load_query_as<T, kWide16>(p, an, ar, at, g, qn, qr);
  else load_query_as<T, kVec16>(p, an, ar, at, g, qn, qr);
}

__device__ inline float max3(float a, float b, float c) {  // (fmaxf first quiets every operand: two instructions more)
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// One lane's half of its query's row: the output, or the part of it over one split's keys.
__device__ inline void store_rows(const PromptProblem& p, int64_t token, int h, int part, int g, f32x16 (&o)[4], float m,
                                  float l) {
  l = sum_halves(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  settle2(o[0], o[1]);
  settle2(o[2], o[3]);
  const int64_t row = token * p.nh + h;
  const bool whole = p.splits == 1;
  float* const po = whole ? nullptr : p.part_o + (int64_t)part * p.q.tokens * p.nh * 128;
  if (whole && p.out_dtype != LA_DTYPE_F32) {
    // 16 B per lane, the halves' middle pieces exchanged
    uint4* const out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * 128);
    const bool bf16 = p.out_dtype == LA_DTYPE_BF16;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int e8 = 0; e8 < 2; ++e8) {
        uint2 w[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = o[d][8 * e8 + 4 * k + e] * inv;
          w[k] = bf16 ? __builtin_bit_cast(uint2, __builtin_convertvector(v, bf16x4))
                      : __builtin_bit_cast(uint2, __builtin_convertvector(v, f16x4));
        }
        const auto x = __builtin_amdgcn_permlane32_swap(w[0].x, w[1].x, false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(w[0].y, w[1].y, false, false);
        out[4 * d + 2 * e8 + g] = uint4{x[0], y[0], x[1], y[1]};
      }
    return;
  }
  float* const to = whole ? static_cast<float*>(p.out) : po;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = o[d][4 * e4 + e] * inv;
      *reinterpret_cast<f32x4*>(to + row * 128 + 32 * d + 8 * e4 + 4 * g) = v;
    }
  if (!whole && g == 0) p.part_lse[(int64_t)part * p.q.tokens * p.nh + row] = l == 0.f ? -INFINITY : m + log2f(l);
}

// What one wave holds of its 32 queries. Scores come out transposed (keys in
// registers, a query per lane), so the softmax's maximum and sum are per lane
// (and one exchange between the lane halves), and their exponentials are the
// second product's operand as they are.
template <typename T>
struct Wave {
  typedef typename Mm<T>::vec vec;
  typedef typename Mm<T>::elem elem;
  typedef const __attribute__((address_space(3))) vec lvec;
  vec qn[8], qr[4];
  vec w[3][4];  // operands of four products, and of the next eight
  f32x16 x[2];  // scores of a tile, less m
  vec pr[4];    // their exponentials
  f32x16 o[4];
  float m, l;   // running maximum, in base-2 units of the scaled scores; sum over this lane half's keys
  f32x16 start; // -m: the scores' sums begin with it, so no instruction subtracts it

  __device__ inline void clear() {
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = f32x16{};
    start = f32x16{};
    m = l = 0.f;
  }
  // Operand k of group i: groups 0..3 are V (group = step of 16 keys, k = block
  // of 32 dims), 4..9 the keys (steps 2 (i - 4) + k / 2, key block k % 2).
  static __device__ inline vec operand(const lchar* b, int i, int k) {
    if (i < 4) return *reinterpret_cast<lvec*>(b + kTileKBytes + 1024 * (4 * k + i));
    const int st = 2 * (i - 4) + (k >> 1), kb = k & 1;
    return *reinterpret_cast<lvec*>(b + (st < 8 ? 1024 * (8 * kb + st) : 2 * kTileKBytes + 1024 * (4 * kb + st - 8)));
  }
  __device__ inline void read(const lchar* b, int i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) w[i % 3][k] = operand(b, i, k);
  }
  // Groups kFrom .. kTo - 1, the operands of each read two groups ahead (those
  // of the first two are there). V comes from tile bv, keys from bk.
  template <int kFrom, int kTo>
  __device__ inline void products(const lchar* bv, const lchar* bk) {
    if constexpr (kTo > 4) x[0] = x[1] = start;
#pragma unroll
    for (int i = kFrom; i < kTo; ++i) {
      if (i + 2 < kTo) read(i + 2 < 4 ? bv : bk, i + 2);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int st = 2 * (i - 4) + (k >> 1);
        if (i < 4) o[k] = Mm<T>::mma(w[i % 3][k], pr[i & 3], o[k]);
        else x[k & 1] = Mm<T>::mma(w[i % 3][k], st < 8 ? qn[st & 7] : qr[st & 3], x[k & 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // Scores -> exponentials. masked: the tile has keys that a token does not see,
  // from number `see` (less 4 per lane half) on. first: the first tile, which
  // sets the maximum whatever it is; later ones raise it where theirs is larger
  // by more than the slack (rarely).
  __device__ inline void softmax(bool masked, int see, bool first) {
    settle2(x[0], x[1]);
    if (masked) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[kb][e] = 32 * kb + 8 * (e >> 2) + (e & 3) < see ? x[kb][e] : -INFINITY;
    }
    float a = max3(x[0][0], x[0][1], x[0][2]), b = max3(x[1][0], x[1][1], x[1][2]);
#pragma unroll
    for (int e = 3; e < 15; e += 2) {
      a = max3(a, x[0][e], x[0][e + 1]);
      b = max3(b, x[1][e], x[1][e + 1]);
    }
    a = max3(a, x[0][15], x[1][15]);
    a = max3(a, b, b);
    const auto sw = __builtin_amdgcn_permlane32_swap(u_of(a), u_of(a), false, false);
    const float top = max3(f_of(sw[0]), f_of(sw[1]), f_of(sw[1]));  // less m
    if (first || __builtin_amdgcn_ballot_w64(top > kSlack)) {
      const float up = first ? (top == -INFINITY ? 0.f : top) : fmaxf(top, 0.f), f = exp2f(-up);
      m += up;
      if (!first) l *= f;  // (f may be infinite then)
      settle2(o[0], o[1]);
      settle2(o[2], o[3]);
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (!first) o[d][e] *= f;
          start[e] = -m;
        }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[kb][e] -= up;
    }
    float sum[4] = {};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_amdgcn_exp2f(x[ks >> 1][8 * (ks & 1) + e]);
        sum[e & 3] += v;
        pr[ks][e] = (elem)v;
      }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }
};

// A workgroup's share of the work: kQBlock tokens of one sequence, one head, one
// of `splits` parts of the keys that they see.
struct Item {
  QueryTile q;
  int h, part, t0, t1;  // head of this launch; key tiles [t0, t1) of the sequence
  const char *kx, *vx, *rx;
};
__device__ inline bool find_item(const PromptProblem& p, Item& it) {
  // An eighth of the items to each XCD, so that the workgroups that read one
  // head's keys share an L2: groups of its heads (every eighth), within them the
  // last query tiles, with the most keys to see, of all heads first. Without
  // groups: an eighth of all, in order of head, part and query tile.
  const int64_t items = (int64_t)p.heads * p.splits * p.q_tiles, per = (items + 7) / 8;
  if ((int64_t)(blockIdx.x >> 3) >= per) return false;
  int qt;
  if (p.group) {
    const uint32_t group = (uint32_t)p.group, one = group * (uint32_t)p.splits * (uint32_t)p.q_tiles;
    const uint32_t k = blockIdx.x >> 3, first = k / one, rest = k - first * one, t = rest / group;
    it.h = (int)((first * group + rest - t * group) * 8 + (blockIdx.x & 7));
    const uint32_t r = t / (uint32_t)p.splits;
    it.part = (int)(t - r * (uint32_t)p.splits);
    qt = (int)((uint32_t)p.q_tiles - 1 - r);
  } else {
    const int64_t item = (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (item >= items) return false;
    const uint32_t qts = (uint32_t)p.q_tiles, hs = (uint32_t)item / qts;
    qt = (int)(qts - 1 - ((uint32_t)item - hs * qts));
    it.part = (int)(hs % (uint32_t)p.splits);
    it.h = (int)(hs / (uint32_t)p.splits);
  }
  if (p.q_info) it.q = p.q_info[qt];
  else it.q = QueryTile{qt * kQBlock, (int)p.q.tokens, p.src.region, p.src.region, 0, 0};
  if (it.q.j0 < 0) return false;
  const int most = tile_visible(it.q, min(it.q.j0 + kQBlock, it.q.n) - 1);  // visible keys grow with the token
  const int nt = (int)clamp64((most + kTileKeys - 1) / kTileKeys, 0, p.src.num_tiles - it.q.tile0);
  it.t0 = (int)((int64_t)nt * it.part / p.splits);
  it.t1 = (int)((int64_t)nt * (it.part + 1) / p.splits);
  const int64_t at = (int64_t)it.h * p.src.num_tiles + it.q.tile0;
  it.kx = static_cast<const char*>(p.kx) + at * kTileKBytes;
  it.vx = static_cast<const char*>(p.vx) + at * kTileKBytes;
  it.rx = static_cast<const char*>(p.rope) + it.q.tile0 * kTileRBytes;
  return true;
}
// HBM -> LDS copy of kPieces KB, 1 KB per instruction, as they lie (an
// instruction's offset moves both addresses). Inline asm without outputs: with
// the builtin the compiler takes every LDS read behind it to be out of order
// and waits for all of them where it needs one (8192 tokens x 128 heads, a call:
// 3018 us so, 2828 with these). It does not count these copies either: landed()
// waits for them.
template <int kPieces>
__device__ inline void copy_run(lchar* to, const char* from, int lane) {
  const uint32_t dst = (uint32_t)(uintptr_t)to, off = 16 * lane;
  static_assert(kPieces == 2 || kPieces == 4, "");
  if constexpr (kPieces == 4)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3\n\t"
                 "global_load_lds_dwordx4 %1, %2 offset:%4\n\tglobal_load_lds_dwordx4 %1, %2 offset:%5"
                 ::"s"(dst), "v"(off), "s"(from), "i"(1 << 10), "i"(2 << 10), "i"(3 << 10) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3"
                 ::"s"(dst), "v"(off), "s"(from), "i"(1 << 10) : "memory", "m0");
}
// Tile t into a buffer: K, V and the rope keys, a quarter of each per wave.
__device__ inline void copy_tile(const Item& it, lchar* b, int t, int wave, int lane) {
  const int c = kTileKBytes / 4 * wave, r = kTileRBytes / 4 * wave;
  copy_run<4>(b + c, it.kx + (int64_t)t * kTileKBytes + c, lane);
  copy_run<4>(b + kTileKBytes + c, it.vx + (int64_t)t * kTileKBytes + c, lane);
  copy_run<2>(b + 2 * kTileKBytes + r, it.rx + (int64_t)t * kTileRBytes + r, lane);
}
__device__ inline void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// 4 waves of 32 tokens over 64 keys at a time, two buffers of 40 KB, two
// workgroups per CU, whose waves overlap each other's softmax and products.
// Bound by its products and, through them, by power: 8192 tokens x 128 heads,
// 2.75 TFLOP, take 2.26 ms, 1.22 PFLOP/s, the matrix cores 69 % busy at the 1.70
// GHz that the card then holds (a whole call 2.54 ms with random numbers, 1.91
// with zeros). Every operand byte serves 32 tokens, so LDS reads (40 KB per wave
// and tile) take as long as the products do; they and the vector work hide
// behind the other waves. Not taken, a call (2743 us then): two groups of four
// waves in step, one in its products while the other is in its softmax, 2716 to
// 2772; 64 tokens per wave, half the reads but one wave per SIMD, 2960 to 3160.
// 64 tokens of one step over 8192 shared rows: 537 MB of keys and values in 107
// us, 5.0 TB/s.
// Roundings to 16 bits, the products' operand type: expanded keys and values,
// the queries (rotated first) and a tile's exponentials, as the decode kernels
// round rows, queries and exponentials; scores, maxima, sums and outputs are
// fp32. The scale goes into one side before its rounding, and the running
// maximum lets exponentials reach 2^8, which fp16 holds.
template <typename T>
__global__ __launch_bounds__(256, 2) void prompt_kernel(PromptProblem p) {
  extern __shared__ __attribute__((aligned(1024))) char prompt_lds[];
  lchar* const lds = (lchar*)prompt_lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int r32 = lane & 31, g = lane >> 5;
  Item it;
  if (!find_item(p, it)) return;
  const int jw = it.q.j0 + kQRows * wave;  // this wave's first token
  const int j = min(jw + r32, it.q.n - 1);
  const int lim = tile_visible(it.q, j);
  const int wave_max = jw < it.q.n ? tile_visible(it.q, min(jw + kQRows, it.q.n) - 1) : 0;
  const int wave_min = tile_visible(it.q, min(jw, it.q.n - 1));
  if (it.t0 < it.t1) copy_tile(it, lds + (it.t0 & 1) * kBufBytes, it.t0, wave, lane);
  const int64_t token = it.q.token0 + j;
  Wave<T> w;
  load_query<T>(p, token, p.head0 + it.h, clamp64(it.q.L - it.q.n + j, 0, INT32_MAX), g, w.qn, w.qr);
  w.clear();
  for (int t = it.t0; t < it.t1; ++t) {
    landed();  // this wave's copies of tile t
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // everyone's; tile t - 1 is read
    if (t + 1 < it.t1) copy_tile(it, lds + ((t + 1) & 1) * kBufBytes, t + 1, wave, lane);
    if (t * kTileKeys >= wave_max) continue;
    const lchar* const b = lds + (t & 1) * kBufBytes + 16 * lane;
    w.read(b, 4);
    w.read(b, 5);
    __builtin_amdgcn_s_setprio(1);  // products first: the other wave of the SIMD has vector work in their shadow
    w.template products<4, 10>(b, b);
    __builtin_amdgcn_s_setprio(0);
    w.read(b, 0);
    w.read(b, 1);
    __builtin_amdgcn_sched_barrier(0);
    w.softmax((t + 1) * kTileKeys > wave_min, lim - t * kTileKeys - 4 * g, t == it.t0);
    __builtin_amdgcn_s_setprio(1);
    w.template products<0, 4>(b, b);
    __builtin_amdgcn_s_setprio(0);
  }
  if (jw + r32 < it.q.n) store_rows(p, token, p.head0 + it.h, it.part, g, w.o, w.m, w.l);
}

template <typename T>
hipError_t prompt_t(const PromptProblem& p, hipStream_t stream) {
  constexpr int lds = 2 * kBufBytes;
  static OncePerDevice once;
  const hipError_t e = allow_lds(once, reinterpret_cast<const void*>(prompt_kernel<T>), lds);
  if (e != hipSuccess) return e;
  const int64_t items = (int64_t)p.heads * p.splits * p.q_tiles;
  if (items > kMostPromptItems) return hipErrorInvalidValue;
  hipLaunchKernelGGL(prompt_kernel<T>, dim3((unsigned)(8 * ((items + 7) / 8))), dim3(256), lds, stream, p);
  return hipGetLastError();
}

// ---- the plain form: any type and head shape ------------------------------------------------------

// One workgroup of 4 waves per (token, head), from number first on, over absorbed fp32 queries: wave w
// takes rows w, w + 4, ... with a running maximum of its own, lanes share a
// row's elements; the waves' sums are joined and projected by W_UV. Everything
// fp32. Rows come from L2 once per head and token, which bounds it; it is there
// for shapes and types that the others do not take.
constexpr int kGenericLatent = 1024;  // kv_lora_rank at most: 16 elements per lane
constexpr int kGenericRope = 256;
__global__ __launch_bounds__(256) void generic_prompt_kernel(GenericPrompt p, int64_t first) {
  __shared__ float q_l[kGenericRope];
  __shared__ float acc_l[4][kGenericLatent];
  __shared__ float ml[4][2];
  const uint32_t item = (uint32_t)first + blockIdx.x;  // (tokens x heads stay below 2^31)
  const int64_t token = item / p.nh;
  const int h = (int)(item % p.nh);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int s = query_seq(p.q, token);
  const int n = query_count(p.q, s);
  const int64_t j = token - query_begin(p.q, s);
  const int L = j >= 0 && j < n ? source_rows(p.src, s) : 0;  // malformed offsets leave tokens without a sequence
  const int keys = L > 0 ? visible_keys(p.q, s, (int)j, n, L) : 0;
  const int half = p.dR / 2;
  const int64_t ar = token * p.q.rope_stride + h * p.q.rope_head;
  const int64_t at = L == 0 ? 0 : source_rope_row(p.src, clamp64(L - n + j, 0, INT32_MAX)) * half;
  for (int i = threadIdx.x; i < half; i += 256) {
    float a = load_any(p.q.q_rope, p.q.dtype, ar + i), b = load_any(p.q.q_rope, p.q.dtype, ar + i + half);
    if (p.q.rotate) {
      const float c = p.src.cos[at + i], sn = p.src.sin[at + i], x = a, y = b;
      a = x * c - y * sn;
      b = x * sn + y * c;
    }
    q_l[i] = a;
    q_l[i + half] = b;
  }
  const float* qa = p.q_abs + ((int64_t)token * p.nh + h) * p.dc;
  float q[16], acc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    q[i] = lane + 64 * i < p.dc ? qa[lane + 64 * i] : 0.f;
    acc[i] = 0.f;
  }
  __syncthreads();
  float m = kNoScore, l = 0.f;
  for (int k = wave; k < keys; k += 4) {
    const int64_t row = source_row(p.src, s, k) * p.src.row_elems;
    float c[16], d = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      c[i] = lane + 64 * i < p.dc ? load_any(p.src.kv, p.src.kv_dtype, row + lane + 64 * i) : 0.f;
      d += q[i] * c[i];
    }
    const int64_t rk = source_rope_row(p.src, k) * half;
    for (int i = lane; i < half; i += 64) {
      const float k0 = load_any(p.src.kv, p.src.kv_dtype, row + p.dc + i);
      const float k1 = load_any(p.src.kv, p.src.kv_dtype, row + p.dc + i + half);
      const float cs = p.src.cos[rk + i], sn = p.src.sin[rk + i];
      d += q_l[i] * (k0 * cs - k1 * sn) + q_l[i + half] * (k0 * sn + k1 * cs);
    }
    const float x = wave_sum(d) * p.scale_log2;
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
    d = wave_sum(d);
    if (lane == 0) store1(p.out, p.out_dtype, ((int64_t)token * p.nh + h) * p.dv + v, keys > 0 ? d : 0.f);
  }
}

// ---- queries of the absorbed forms ------------------------------------------------------------------

// kTokenElems elements of a token's nope queries, and as many pairs of rope
// ones, per workgroup (x: token from number token0 on, y: share), four at a time where heads and
// strides are whole vectors; the first also writes its length and table.
constexpr int kTokenElems = 2048;
template <int kN>
__device__ inline void load_n(const void* base, int dtype, int64_t i, float (&x)[kN]) {
  if constexpr (kN == 4) load_q4(base, dtype, i, x);
  else x[0] = load_any(base, dtype, i);
}
template <int kN>
__global__ __launch_bounds__(256) void tokens_kernel(TokenProblem p, int64_t token0) {
  const int64_t token = token0 + blockIdx.x;
  const int s = query_seq(p.q, token);
  const int n = query_count(p.q, s);
  const int64_t j = token - query_begin(p.q, s);
  const int L = j >= 0 && j < n ? source_rows(p.src, s) : 0;  // malformed offsets leave tokens without a sequence
  const int first = blockIdx.y * kTokenElems + kN * threadIdx.x, last = (blockIdx.y + 1) * kTokenElems;
  if (p.lens && first == 0) p.lens[token] = L > 0 ? visible_keys(p.q, s, (int)j, n, L) : 0;
  if (p.table && blockIdx.y == 0) {
    int32_t* const t = p.table + token * p.blocks_per_seq;
    for (int i = threadIdx.x; i < p.blocks_per_seq; i += 256)
      t[i] = L == 0 || i >= p.used_blocks ? 0
             : p.src.block_table         ? p.src.block_table[(int64_t)s * p.src.blocks_per_seq + i]
                                         : (int32_t)((int64_t)s * p.src.stride_rows / p.block_size + i);
  }
  if (p.q_nope)
    for (int i = first; i < min(p.nh * p.dn, last); i += 256 * kN) {
      float x[kN];
      load_n<kN>(p.q.q_nope, p.q.dtype, token * p.q.nope_stride + (i / p.dn) * p.q.nope_head + i % p.dn, x);
#pragma unroll
      for (int e = 0; e < kN; ++e) p.q_nope[token * p.nh * p.dn + i + e] = x[e];
    }
  if (p.q_rope) {
    const int half = p.dR / 2;
    const int64_t at = L == 0 ? 0 : source_rope_row(p.src, clamp64(L - n + j, 0, INT32_MAX)) * half;
    for (int i = first; i < min(p.nh * half, last); i += 256 * kN) {
      const int h = i / half, d = i % half;
      const int64_t ar = token * p.q.rope_stride + h * p.q.rope_head + d;
      float a[kN], b[kN];
      load_n<kN>(p.q.q_rope, p.q.dtype, ar, a);
      load_n<kN>(p.q.q_rope, p.q.dtype, ar + half, b);
      float* const o = p.q_rope + (token * p.nh + h) * p.dR + d;
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float x = a[e], y = b[e];
        if (p.q.rotate) {
          const float c = p.src.cos[at + d + e], sn = p.src.sin[at + d + e];
          a[e] = x * c - y * sn;
          b[e] = x * sn + y * c;
        }
        o[e] = a[e];
        o[half + e] = b[e];
      }
    }
  }
}

__global__ __launch_bounds__(256) void cast_kernel(const float* src, void* dst, int out_dtype, int64_t n) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step) store1(dst, out_dtype, i, src[i]);
}

}  // namespace

int prompt_query_rows() { return kQBlock; }

hipError_t launch_prompt(const PromptProblem& p, hipStream_t stream) {
  if (p.q_tiles == 0 || p.heads == 0) return hipSuccess;
  return p.f16 ? prompt_t<__half>(p, stream) : prompt_t<__hip_bfloat16>(p, stream);
}

bool generic_prompt_supported(int dc, int dR) { return dc <= kGenericLatent && dR <= kGenericRope; }

hipError_t launch_generic_prompt(const GenericPrompt& p, hipStream_t stream) {
  const int64_t items = p.q.tokens * p.nh;
  if (items > INT32_MAX) return hipErrorInvalidValue;
  return in_grids(items, most_blocks(256), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL(generic_prompt_kernel, dim3(blocks), dim3(256), 0, stream, p, first);
  });
}

hipError_t launch_tokens(const TokenProblem& p, hipStream_t stream) {
  const int elems = p.nh * (p.dn > p.dR / 2 ? p.dn : p.dR / 2);
  const unsigned shares = (unsigned)((elems + kTokenElems - 1) / kTokenElems);
  if (shares > kMostBlocksYZ) return hipErrorInvalidValue;
  const auto k = p.vec && p.dn % 4 == 0 && p.dR % 8 == 0 ? tokens_kernel<4> : tokens_kernel<1>;
  return in_grids(p.q.tokens, most_blocks(256), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL(k, dim3(blocks, shares), dim3(256), 0, stream, p, first);
  });
}

hipError_t launch_cast(const float* src, void* dst, int out_dtype, int64_t n, hipStream_t stream) {
  if (n == 0) return hipSuccess;
  const int64_t blocks = n / 1024 + 1 < 4096 ? n / 1024 + 1 : 4096;
  hipLaunchKernelGGL(cast_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, src, dst, out_dtype, n);
  return hipGetLastError();
}

}  // namespace la
