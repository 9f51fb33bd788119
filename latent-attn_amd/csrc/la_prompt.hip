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
typedef __attribute__((address_space(3))) void lds_void;
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

__device__ inline void store4(void* out, int dtype, int64_t i, f32x4 v) {
  if (dtype == LA_DTYPE_F32) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(out) + i) = v;
  } else if (dtype == LA_DTYPE_BF16) {
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<v4*>(static_cast<__bf16*>(out) + i) = __builtin_convertvector(v, v4);
  } else {
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<v4*>(static_cast<_Float16*>(out) + i) = __builtin_convertvector(v, v4);
  }
}
__device__ inline void store1(void* out, int dtype, int64_t i, float v) {
  if (dtype == LA_DTYPE_F32) static_cast<float*>(out)[i] = v;
  else if (dtype == LA_DTYPE_BF16) static_cast<__bf16*>(out)[i] = (__bf16)v;
  else static_cast<_Float16*>(out)[i] = (_Float16)v;
}

// The query of one lane as operands: 12 steps of 8 elements, step by step {16 k +
// 4 g + (0..3), 16 k + 8 + 4 g + (0..3)}. All loads go out before the first is
// waited for, so the type decides around them, not between them.
enum QueryLoad { kScalar, kVec16, kVec32 };
template <typename T, QueryLoad kLoad>
__device__ inline void load_query_as(const PromptProblem& p, int64_t an, int64_t ar, int64_t pos, int g,
                                     typename Mm<T>::vec (&qn)[8], typename Mm<T>::vec (&qr)[4]) {
  typedef typename Mm<T>::elem elem;
  float x[24][4];  // 16 pieces of the nope part, 8 of the rope part
  auto at = [&](int i) { return i < 16 ? an + 8 * i + 4 * g : ar + 8 * (i - 16) + 4 * g; };
  if constexpr (kLoad == kVec16) {
    uint2 w[24];
#pragma unroll
    for (int i = 0; i < 24; ++i)
      w[i] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(i < 16 ? p.q.q_nope : p.q.q_rope) + at(i));
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
      if (i < 16) qn[i >> 1][4 * (i & 1) + e] = (elem)x[i][e];
      else qr[(i - 16) >> 1][4 * (i & 1) + e] = (elem)x[i][e];
    }
}
template <typename T>
__device__ inline void load_query(const PromptProblem& p, int64_t token, int h, int64_t pos, int g,
                                  typename Mm<T>::vec (&qn)[8], typename Mm<T>::vec (&qr)[4]) {
  const int64_t an = token * p.q.nope_stride + h * p.q.nope_head, ar = token * p.q.rope_stride + h * p.q.rope_head;
  const int64_t at = source_rope_row(p.src, pos) * 32;
  if (!(p.nope_vec && p.rope_vec)) load_query_as<T, kScalar>(p, an, ar, at, g, qn, qr);
  else if (p.q.dtype == LA_DTYPE_F32) load_query_as<T, kVec32>(p, an, ar, at, g, qn, qr);
  else load_query_as<T, kVec16>(p, an, ar, at, g, qn, qr);
}

// One workgroup: kQBlock tokens of one sequence, one head, one of `splits`
// parts of the keys that they see. Scores come out transposed (keys in
// registers, a query per lane), so the softmax's maximum and sum are per lane
// (and one exchange between the lane halves), and their exponentials are the
// second product's operand as they are.
template <typename T>
__global__ __launch_bounds__(256, 2) void prompt_kernel(PromptProblem p) {
  typedef typename Mm<T>::vec vec;
  typedef typename Mm<T>::elem elem;
  extern __shared__ __attribute__((aligned(1024))) char prompt_lds[];
  lchar* const lds = (lchar*)prompt_lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int r32 = lane & 31, g = lane >> 5;
  // Items in order of head, part and query tile (the last, with the most keys
  // to see, first), an eighth of them to each XCD: the workgroups that read
  // one head's keys share an L2.
  const int64_t items = (int64_t)p.heads * p.splits * p.q_tiles, per = (items + 7) / 8;
  const int64_t item = (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int64_t)(blockIdx.x >> 3) >= per || item >= items) return;
  const int64_t qt = p.q_tiles - 1 - item % p.q_tiles;
  const int hs = (int)(item / p.q_tiles), part = hs % p.splits, h = hs / p.splits;
  QueryTile q;
  if (p.q_info) q = p.q_info[qt];
  else q = QueryTile{(int)qt * kQBlock, (int)p.q.tokens, p.src.region, p.src.region, 0, 0};
  if (q.j0 < 0) return;
  // visible keys grow with the token
  const int jw = q.j0 + kQRows * wave;  // this wave's first token
  const int j = min(jw + r32, q.n - 1);
  const int lim = tile_visible(q, j);
  const int wave_max = jw < q.n ? tile_visible(q, min(jw + kQRows, q.n) - 1) : 0;
  const int wave_min = tile_visible(q, min(jw, q.n - 1));
  const int block_max = tile_visible(q, min(q.j0 + kQBlock, q.n) - 1);
  const int64_t tile0 = q.tile0;
  const int nt = (int)clamp64((block_max + kTileKeys - 1) / kTileKeys, 0, p.src.num_tiles - tile0);
  const int t0 = (int)((int64_t)nt * part / p.splits), t1 = (int)((int64_t)nt * (part + 1) / p.splits);

  const char* const kx = static_cast<const char*>(p.kx) + ((int64_t)h * p.src.num_tiles + tile0) * kTileKBytes;
  const char* const vx = static_cast<const char*>(p.vx) + ((int64_t)h * p.src.num_tiles + tile0) * kTileKBytes;
  const char* const rx = static_cast<const char*>(p.rope) + tile0 * kTileRBytes;
  // A tile is three runs of 16, 16 and 8 KB, copied as they lie: 1 KB per wave and instruction.
  auto issue = [&](int t) {
    lchar* const b = lds + (t & 1) * kBufBytes;
    const char* k = kx + (int64_t)t * kTileKBytes + 16 * lane;
    const char* v = vx + (int64_t)t * kTileKBytes + 16 * lane;
    const char* r = rx + (int64_t)t * kTileRBytes + 16 * lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 1024 * (4 * i + wave);
      __builtin_amdgcn_global_load_lds(k + c, (lds_void*)(b + c), 16, 0, 0);
      __builtin_amdgcn_global_load_lds(v + c, (lds_void*)(b + kTileKBytes + c), 16, 0, 0);
      if (i < 2) __builtin_amdgcn_global_load_lds(r + c, (lds_void*)(b + 2 * kTileKBytes + c), 16, 0, 0);
    }
  };
  if (t0 < t1) issue(t0);

  const int64_t token = q.token0 + j;
  vec qn[8], qr[4];
  load_query<T>(p, token, p.head0 + h, clamp64(q.L - q.n + j, 0, INT32_MAX), g, qn, qr);

  f32x16 o[4] = {};
  float m = kNoScore, l = 0.f;  // m in base-2 units of the scaled scores; l: this lane half's keys
  const float sc = p.scale_log2;
  for (int t = t0; t < t1; ++t) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // this wave's copies of tile t have landed
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // everyone's; tile t - 1 is read
    if (t + 1 < t1) issue(t + 1);
    if (t * kTileKeys >= wave_max) continue;
    const lchar* const b = lds + (t & 1) * kBufBytes + 16 * lane;
    auto operand = [&](int at) { return *reinterpret_cast<const __attribute__((address_space(3))) vec*>(b + at); };
    // products in groups of four, the operands of the next group read before them
    auto key = [&](int i) {  // operand i: step i / 2, key block i % 2
      return operand(i < 16 ? 1024 * (8 * (i & 1) + (i >> 1)) : 2 * kTileKBytes + 1024 * (4 * (i & 1) + (i >> 1) - 8));
    };
    f32x16 x[2] = {};
    vec w[2][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[0][k] = key(k);
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      if (i < 5) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[(i + 1) & 1][k] = key(4 * (i + 1) + k);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int st = (4 * i + k) >> 1;
        x[k & 1] = Mm<T>::mma(w[i & 1][k], st < 8 ? qn[st] : qr[st - 8], x[k & 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    vec v[2][4];
#pragma unroll
    for (int d = 0; d < 4; ++d) v[0][d] = operand(kTileKBytes + 1024 * (4 * d));
    __builtin_amdgcn_sched_barrier(0);
    settle2(x[0], x[1]);
    if ((t + 1) * kTileKeys > wave_min) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          x[kb][e] = t * kTileKeys + 32 * kb + 8 * (e >> 2) + 4 * g + (e & 3) < lim ? x[kb][e] : -INFINITY;
    }
    float top = x[0][0];
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, fmaxf(x[0][e], x[1][e]));
    const auto sw = __builtin_amdgcn_permlane32_swap(u_of(top), u_of(top), false, false);
    top = fmaxf(f_of(sw[0]), f_of(sw[1])) * sc;
    if (__builtin_amdgcn_ballot_w64(top > m + kSlack)) {
      const float up = fmaxf(m, top), a = exp2f(m - up);
      m = up;
      l *= a;
      settle2(o[0], o[1]);
      settle2(o[2], o[3]);
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= a;
    }
    vec pr[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(x[ks >> 1][8 * (ks & 1) + e], sc, -m));
        l += w;
        pr[ks][e] = (elem)w;
      }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks < 3) {
#pragma unroll
        for (int d = 0; d < 4; ++d) v[(ks + 1) & 1][d] = operand(kTileKBytes + 1024 * (4 * d + ks + 1));
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] = Mm<T>::mma(v[ks & 1][d], pr[ks], o[d]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (jw + r32 >= q.n) return;
  l = sum_halves(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  settle2(o[0], o[1]);
  settle2(o[2], o[3]);
  const int64_t row = token * p.nh + p.head0 + h;
  const bool whole = p.splits == 1;
  float* const po = whole ? nullptr : p.part_o + (int64_t)part * p.q.tokens * p.nh * 128;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = o[d][4 * e4 + e] * inv;
      const int64_t at = row * 128 + 32 * d + 8 * e4 + 4 * g;
      if (whole) store4(p.out, p.out_dtype, at, v);
      else *reinterpret_cast<f32x4*>(po + at) = v;
    }
  if (!whole && g == 0) p.part_lse[(int64_t)part * p.q.tokens * p.nh + row] = l == 0.f ? -INFINITY : m + log2f(l);
}

template <typename T>
hipError_t prompt_t(const PromptProblem& p, hipStream_t stream) {
  constexpr int lds = 2 * kBufBytes;
  static OncePerDevice once;
  hipError_t e = allow_lds(once, reinterpret_cast<const void*>(prompt_kernel<T>), lds);
  if (e != hipSuccess) return e;
  const int64_t items = (int64_t)p.heads * p.splits * p.q_tiles;
  if (items > INT32_MAX - 8) return hipErrorInvalidValue;
  hipLaunchKernelGGL(prompt_kernel<T>, dim3((unsigned)(8 * ((items + 7) / 8))), dim3(256), lds, stream, p);
  return hipGetLastError();
}

// ---- the plain form: any type and head shape ------------------------------------------------------

// One workgroup of 4 waves per (token, head) over absorbed fp32 queries: wave w
// takes rows w, w + 4, ... with a running maximum of its own, lanes share a
// row's elements; the waves' sums are joined and projected by W_UV.
constexpr int kGenericLatent = 1024;  // kv_lora_rank at most: 16 elements per lane
constexpr int kGenericRope = 256;
__global__ __launch_bounds__(256) void generic_prompt_kernel(GenericPrompt p) {
  __shared__ float q_l[kGenericRope];
  __shared__ float acc_l[4][kGenericLatent];
  __shared__ float ml[4][2];
  const int64_t token = blockIdx.x / p.nh;
  const int h = (int)(blockIdx.x % p.nh);
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

// kTokenElems elements of a token's queries per workgroup (x: token, y: share);
// the first also writes its length and table.
constexpr int kTokenElems = 2048;
__global__ __launch_bounds__(256) void tokens_kernel(TokenProblem p) {
  const int64_t token = blockIdx.x;
  const int s = query_seq(p.q, token);
  const int n = query_count(p.q, s);
  const int64_t j = token - query_begin(p.q, s);
  const int L = j >= 0 && j < n ? source_rows(p.src, s) : 0;  // malformed offsets leave tokens without a sequence
  const int first = blockIdx.y * kTokenElems + threadIdx.x, last = (blockIdx.y + 1) * kTokenElems;
  if (p.lens && first == 0) p.lens[token] = L > 0 ? visible_keys(p.q, s, (int)j, n, L) : 0;
  if (p.table && blockIdx.y == 0) {
    int32_t* const t = p.table + token * p.blocks_per_seq;
    for (int i = threadIdx.x; i < p.blocks_per_seq; i += 256)
      t[i] = L == 0                 ? 0
             : p.src.block_table ? p.src.block_table[(int64_t)s * p.src.blocks_per_seq + i]
                                 : (int32_t)((int64_t)s * p.src.stride_rows / p.block_size + i);
  }
  if (p.q_nope)
    for (int i = first; i < min(p.nh * p.dn, last); i += 256)
      p.q_nope[token * p.nh * p.dn + i] =
          load_any(p.q.q_nope, p.q.dtype, token * p.q.nope_stride + (i / p.dn) * p.q.nope_head + i % p.dn);
  if (p.q_rope) {
    const int half = p.dR / 2;
    const int64_t at = L == 0 ? 0 : source_rope_row(p.src, clamp64(L - n + j, 0, INT32_MAX)) * half;
    for (int i = first; i < min(p.nh * half, last); i += 256) {
      const int h = i / half, d = i % half;
      const int64_t ar = token * p.q.rope_stride + h * p.q.rope_head + d;
      float a = load_any(p.q.q_rope, p.q.dtype, ar), b = load_any(p.q.q_rope, p.q.dtype, ar + half);
      if (p.q.rotate) {
        const float c = p.src.cos[at + d], sn = p.src.sin[at + d], x = a, y = b;
        a = x * c - y * sn;
        b = x * sn + y * c;
      }
      float* const o = p.q_rope + (token * p.nh + h) * p.dR + d;
      o[0] = a;
      o[half] = b;
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
  const int64_t blocks = p.q.tokens * p.nh;
  if (blocks == 0) return hipSuccess;
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL(generic_prompt_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_tokens(const TokenProblem& p, hipStream_t stream) {
  if (p.q.tokens == 0) return hipSuccess;
  if (p.q.tokens > INT32_MAX) return hipErrorInvalidValue;
  const int elems = p.nh * (p.dn > p.dR / 2 ? p.dn : p.dR / 2);
  const unsigned shares = (unsigned)((elems + kTokenElems - 1) / kTokenElems);
  if (shares > 65535) return hipErrorInvalidValue;
  hipLaunchKernelGGL(tokens_kernel, dim3((unsigned)p.q.tokens, shares), dim3(256), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_cast(const float* src, void* dst, int out_dtype, int64_t n, hipStream_t stream) {
  if (n == 0) return hipSuccess;
  const int64_t blocks = n / 1024 + 1 < 4096 ? n / 1024 + 1 : 4096;
  hipLaunchKernelGGL(cast_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, src, dst, out_dtype, n);
  return hipGetLastError();
}

}  // namespace la
