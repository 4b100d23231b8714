// Rotary positions on several axes (time, height, width, ...), with the RMS norm of q and k in front.
//
//   angle[token, j] = position[token, axis(j)] * inv_freq[j]           j = 0 .. pairs-1, axis(j) from the sections
//   (u, v) of pair j of every head -> (u cos - v sin, u sin + v cos)
//
// Pairs are neighbours (2j, 2j+1) or half the rotated length apart (j, j + pairs); elements past 2 * pairs pass through.
// The angle is reduced in 64 bits (a turn is position * inv_freq / 2 pi less its nearest whole number), so positions in the
// millions keep the full 32-bit sine and cosine; computed once per token and shared by all its heads through shared
// memory, that costs a fraction of a percent of the kernel, which is bound by HBM: q and k are read once and written
// once.  No table of sines: any position is served, a fraction or a negative one too.
//
// A block takes some tokens; a head is covered by `lanes` lanes (a power of two), each with a chunk of it: 8 neighbouring
// elements (4 pairs), or - pairs half a head apart - 8 or 4 neighbours and their partners, so that no lane needs another's
// elements (pairs no multiple of 4: 8 of them, element by element).  The kernel is near its issue slots besides HBM: the
// weights of the head norm are multiplied into the token's table of turns (once per token instead of once per head), and a
// lane's loads of several heads are issued before the first is used.  The norm over a token's heads reads a token that does
// not fit its block's registers twice, the second time out of the L1.
#include "sq_internal.h"
#include "sq_overlap.h"
#include "sq_rows.cuh"

namespace sq {
namespace {

struct RotaryArgs {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int64_t q_in[2], k_in[2], q_to[2], k_to[2];      // strides in elements: batch, token
  int q_in_head, k_in_head, q_to_head, k_to_head;  // and head
  const void* q_weight;
  const void* k_weight;
  int q_weight_f32, k_weight_f32;
  const void* positions;
  int position_type;
  int64_t position_batch, position_token;  // strides in elements; the axes of a token are neighbours
  const double* inv_freq;
  int section_end[SQ_ROTARY_AXES];
  int64_t length;           // tokens of a batch
  uint32_t blocks_per_batch;
  int heads, kv_heads, dim, pairs;
  int lanes_log2, chunks, tokens_per_block;
  int table_rows;           // of a token's table: a lane's pairs, one row each
  int table_lanes;          // entries of a row
  // n / d as the high word of n * ceil(2^32 / d), exact while n * d < 2^32 (0: d is 1)
  uint32_t heads_magic;     // d = heads + kv_heads up to 4096, items below 2^20
  uint32_t token_magic, row_magic;  // d = a token's table entries, a row's: no more than 512 + 32 entries in all
  float eps, inv_dim;
};

__device__ __forceinline__ double position_at(const RotaryArgs& a, int64_t at) {
  if (a.position_type == SQ_POS_INT32) return static_cast<double>(static_cast<const int32_t*>(a.positions)[at]);
  if (a.position_type == SQ_POS_INT64) return static_cast<double>(static_cast<const int64_t*>(a.positions)[at]);
  return static_cast<double>(static_cast<const float*>(a.positions)[at]);
}

__device__ __forceinline__ float one_param(const void* base, int64_t index, bool f32, const __nv_bfloat16*) {
  return f32 ? __ldg(static_cast<const float*>(base) + index) : __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(base) + index));
}
__device__ __forceinline__ float one_param(const void* base, int64_t index, bool f32, const __half*) {
  return f32 ? __ldg(static_cast<const float*>(base) + index) : __half2float(__ldg(static_cast<const __half*>(base) + index));
}

__device__ __forceinline__ int quotient(int n, uint32_t magic) { return magic == 0 ? n : static_cast<int>(__umulhi(n, magic)); }

// C elements of 16 bits, as loaded
template <int C>
struct Chunk {
  uint32_t w[C / 2];
};
template <int C>
__device__ __forceinline__ Chunk<C> load_chunk(const void* p) {
  Chunk<C> c;
  if constexpr (C == 8)
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(c.w[0]), "=r"(c.w[1]), "=r"(c.w[2]), "=r"(c.w[3]) : "l"(p) : "memory");
  else
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(c.w[0]), "=r"(c.w[1]) : "l"(p) : "memory");
  return c;
}
template <int C>
__device__ __forceinline__ void store_chunk(void* p, const Chunk<C>& c) {
  if constexpr (C == 8) *static_cast<uint4*>(p) = make_uint4(c.w[0], c.w[1], c.w[2], c.w[3]);
  else *static_cast<uint2*>(p) = make_uint2(c.w[0], c.w[1]);
}
// the first `count` of them one by one; the others are zero
template <int C>
__device__ __forceinline__ Chunk<C> load_elements(const void* p, int count) {
  Chunk<C> c;
  const volatile uint16_t* x = static_cast<const volatile uint16_t*>(p);
#pragma unroll
  for (int i = 0; i < C / 2; ++i) {
    const uint32_t lo = 2 * i < count ? x[2 * i] : 0u, hi = 2 * i + 1 < count ? x[2 * i + 1] : 0u;
    c.w[i] = lo | (hi << 16);
  }
  return c;
}
template <int C>
__device__ __forceinline__ void store_elements(void* p, const Chunk<C>& c, int count) {
  uint16_t* x = static_cast<uint16_t*>(p);
#pragma unroll
  for (int e = 0; e < C; ++e)
    if (e < count) x[e] = static_cast<uint16_t>(c.w[e / 2] >> (16 * (e & 1)));
}
template <int C>
__device__ __forceinline__ void widen(const Chunk<C>& c, float (&f)[C], const __nv_bfloat16*) {
#pragma unroll
  for (int i = 0; i < C / 2; ++i) {
    f[2 * i] = __uint_as_float(c.w[i] << 16);
    f[2 * i + 1] = __uint_as_float(c.w[i] & 0xFFFF0000u);
  }
}
template <int C>
__device__ __forceinline__ void widen(const Chunk<C>& c, float (&f)[C], const __half*) {
#pragma unroll
  for (int i = 0; i < C / 2; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&c.w[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, const __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int C, typename T>
__device__ __forceinline__ Chunk<C> narrow(const float (&f)[C], const T* tag) {
  Chunk<C> c;
#pragma unroll
  for (int i = 0; i < C / 2; ++i) c.w[i] = narrow2(f[2 * i], f[2 * i + 1], tag);
  return c;
}

// kHalf: pairs half a head apart.  C: elements of each of a lane's two chunks (interleaved: 4, the halves of 8 neighbours).
// kElement: a lane may hold less than its share of pairs.  Half a head apart: pairs no multiple of C, chunks end short and
// elements move one by one.  Interleaved: pairs past the last turned one do not meet - infinity times the sine of zero would make
// a neighbour NaN (a form of its own, since asking costs 153 us instead of 145 with the head norm, 32768 tokens of 40 heads).
template <typename T, bool kHalf, int C, bool kElement, int kNorm>
__global__ void __launch_bounds__(256) sq_rotary_kernel(const RotaryArgs a) {
  constexpr bool kHead = kNorm == SQ_ROTARY_NORM_HEAD, kToken = kNorm == SQ_ROTARY_NORM_TOKEN;
  constexpr int kAtOnce = 4;  // heads of a lane whose loads are under way together
  extern __shared__ __align__(16) float smem[];
  const T* tag = nullptr;
  // a token's table of turns, a row for each of a lane's pairs: neighbouring lanes read neighbouring entries (with a lane's
  // own entries next to each other its reads collided eight ways in shared memory: 371 us against 159, 32768 tokens of 40 heads)
  const int half = a.table_rows * a.table_lanes;
  // head norm: (wu c, wv s, wu s, wv c) for q, then for k; else (c, s)
  float4* wide = reinterpret_cast<float4*>(smem);
  float2* plain = reinterpret_cast<float2*>(smem);
  float* sums = smem + 2 * a.tokens_per_block * half;  // token norm: [tokens][heads + kv_heads], then 1 / rms [tokens][q, k]

  const int all_heads = a.heads + a.kv_heads;
  const uint32_t batch = blockIdx.x / a.blocks_per_batch;
  const int64_t first_token = static_cast<int64_t>(blockIdx.x - batch * a.blocks_per_batch) * a.tokens_per_block;
  const int here = static_cast<int>(min(static_cast<int64_t>(a.tokens_per_block), a.length - first_token));
  for (int i = threadIdx.x; i < here * half; i += 256) {
    const int token = quotient(i, a.token_magic), entry = i - token * half;
    const int at_row = quotient(entry, a.row_magic), j = (entry - at_row * a.table_lanes) * a.table_rows + at_row;
    float2 cs = make_float2(1.0f, 0.0f);  // interleaved, pairs past `pairs` are not turned
    if (j < a.pairs) {
      int axis = 0;
#pragma unroll
      for (int x = 0; x < SQ_ROTARY_AXES - 1; ++x) axis += j >= a.section_end[x] ? 1 : 0;
      const int64_t at = batch * a.position_batch + (first_token + token) * a.position_token + axis;
      const double turns = position_at(a, at) * a.inv_freq[j] * 0.15915494309189533577;  // 1 / (2 pi)
      const float part = static_cast<float>(turns - rint(turns));
      sincospif(2.0f * part, &cs.y, &cs.x);
    }
    if (kHead) {
      const int u = kHalf ? j : 2 * j, v = kHalf ? j + a.pairs : 2 * j + 1;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const void* w = s ? a.k_weight : a.q_weight;
        const bool f32 = (s ? a.k_weight_f32 : a.q_weight_f32) != 0;
        const bool weighed = w != nullptr && (kHalf ? j < a.pairs : 2 * j < a.dim);
        const float wu = weighed ? one_param(w, u, f32, tag) : 1.0f, wv = weighed ? one_param(w, v, f32, tag) : 1.0f;
        wide[s * a.tokens_per_block * half + i] = make_float4(wu * cs.x, wv * cs.y, wu * cs.y, wv * cs.x);
      }
    } else {
      plain[i] = cs;
    }
  }

  const int lanes = 1 << a.lanes_log2, lane = threadIdx.x & (lanes - 1);
  const int segments = 256 >> a.lanes_log2, items = here * all_heads;
  const T* q = static_cast<const T*>(a.q) + batch * a.q_in[0] + first_token * a.q_in[1];
  const T* k = static_cast<const T*>(a.k) + batch * a.k_in[0] + first_token * a.k_in[1];
  T* q_to = static_cast<T*>(a.q_out) + batch * a.q_to[0] + first_token * a.q_to[1];
  T* k_to = static_cast<T*>(a.k_out) + batch * a.k_to[0] + first_token * a.k_to[1];
  // this lane's two chunks: C pairs (the partners `apart` elements on), or a piece of the tail that is not turned
  const int turned = (a.pairs + C - 1) / C;  // chunks with pairs
  const bool tail = kHalf && lane >= turned;
  const int left = a.pairs - 4 * lane;  // interleaved and kElement: of this lane's four pairs, how many are turned
  const int first = !kHalf ? lane * 8 : tail ? 2 * a.pairs + (lane - turned) * 2 * C : lane * C;
  const int apart = !kHalf ? 4 : tail ? C : a.pairs;
  const bool on = lane < a.chunks, on2 = on && (!tail || first + C < a.dim);
  const int count = tail ? a.dim - first : a.pairs - first, count2 = tail ? count - C : count;  // elements left (kElement)

  struct Item {
    int token, head;
    bool is_q;
  };
  auto decode = [&](int item) {
    Item it;
    it.token = quotient(item, a.heads_magic);
    const int h = item - it.token * all_heads;
    it.is_q = h < a.heads;
    it.head = it.is_q ? h : h - a.heads;
    return it;
  };
  auto source = [&](const Item& it) {
    return it.is_q ? q + it.token * a.q_in[1] + static_cast<int64_t>(it.head) * a.q_in_head
                   : k + it.token * a.k_in[1] + static_cast<int64_t>(it.head) * a.k_in_head;
  };
  auto load = [&](const T* from, Chunk<C>& u, Chunk<C>& v) {
    if (!kHalf) {  // one vector of 8
      const Chunk<8> w = load_chunk<8>(from + first);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u.w[i < C / 2 ? i : 0] = w.w[i];
        v.w[i < C / 2 ? i : 0] = w.w[2 + i];
      }
    } else if (kElement) {
      u = load_elements<C>(from + first, count);
      v = load_elements<C>(from + first + apart, count2);
    } else {
      u = load_chunk<C>(from + first);
      if (on2) v = load_chunk<C>(from + first + apart);
    }
  };
  auto squares = [&](const Chunk<C>& u, const Chunk<C>& v) {
    float s = 0.0f, fu[C], fv[C];
    widen(u, fu, tag);
    widen(v, fv, tag);
#pragma unroll
    for (int e = 0; e < C; ++e) s = fmaf(fu[e], fu[e], fmaf(fv[e], fv[e], s));
    return s;
  };

  float* roots = sums + a.tokens_per_block * all_heads;
  auto join = [&]() {  // 1 / rms of each token's q and k, a warp each
    __syncthreads();
    for (int i = threadIdx.x >> 5; i < 2 * here; i += 8) {
      const int begin = (i & 1) ? a.heads : 0, count_heads = (i & 1) ? a.kv_heads : a.heads;
      float s = 0.0f;
      for (int h = threadIdx.x & 31; h < count_heads; h += 32) s += sums[(i >> 1) * all_heads + begin + h];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if ((threadIdx.x & 31) == 0) roots[i] = __frsqrt_rn(s / (static_cast<float>(count_heads) * static_cast<float>(a.dim)) + a.eps);
    }
  };
  const bool once = items <= kAtOnce * segments;  // the block's items fit its threads' registers: no second reading
  if (kToken && !once) {
    for (int item = threadIdx.x >> a.lanes_log2; item < (items + segments - 1) / segments * segments; item += segments) {
      float s = 0.0f;
      if (item < items && on) {
        Chunk<C> u = {}, v = {};
        load(source(decode(item)), u, v);
        s = squares(u, v);
      }
      for (int d = lanes >> 1; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (lane == 0 && item < items) sums[item] = s;
    }
    join();
  }
  if (!kToken || !once) __syncthreads();

  for (int item0 = threadIdx.x >> a.lanes_log2; item0 < (items + segments - 1) / segments * segments; item0 += kAtOnce * segments) {
    Chunk<C> u[kAtOnce], v[kAtOnce];
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const int item = item0 + n * segments;
#pragma unroll
      for (int i = 0; i < C / 2; ++i) u[n].w[i] = v[n].w[i] = 0;
      if (item < items && on) load(source(decode(item)), u[n], v[n]);
    }
    if (kToken && once) {  // the only round: every thread is here
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        const int item = item0 + n * segments;
        float s = squares(u[n], v[n]);
        for (int d = lanes >> 1; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0 && item < items) sums[item] = s;
      }
      join();
      __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const int item = item0 + n * segments;
      float scale = 1.0f;
      if (kHead) {
        float s = squares(u[n], v[n]);
        for (int d = lanes >> 1; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        scale = rsqrtf(fmaf(s, a.inv_dim, a.eps));  // once per head and lane: the correctly rounded root costs 11 us of 162
      }
      if (item >= items || !on) continue;
      const Item it = decode(item);
      if (kToken) scale = roots[2 * it.token + (it.is_q ? 0 : 1)];
      float fu[C], fv[C];
      widen(u[n], fu, tag);
      widen(v[n], fv, tag);
      if (kNorm != SQ_ROTARY_NORM_NONE) {
#pragma unroll
        for (int e = 0; e < C; ++e) {
          fu[e] *= scale;
          fv[e] *= scale;
        }
      }
      const void* w = it.is_q ? a.q_weight : a.k_weight;
      const bool f32 = (it.is_q ? a.q_weight_f32 : a.k_weight_f32) != 0;
      if ((kToken || (kHead && tail)) && w != nullptr) {
        const int64_t at = (kToken ? static_cast<int64_t>(it.head) * a.dim : 0) + first;
        if (!kHalf) {
          float p[8];
          load_params<T>(w, at, f32, p);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            fu[e < C ? e : 0] *= p[e];
            fv[e < C ? e : 0] *= p[4 + e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < C; ++e) {
            if (!kElement || e < count) fu[e] *= one_param(w, at + e, f32, tag);
            if (on2 && (!kElement || e < count2)) fv[e] *= one_param(w, at + apart + e, f32, tag);
          }
        }
      }
      if (!tail) {
        const int entry = it.token * half + lane;
        if (kHead) {
          const float4* t = wide + (it.is_q ? 0 : a.tokens_per_block * half) + entry;
          if (kHalf) {
#pragma unroll
            for (int e = 0; e < C; ++e) {
              const float4 m = t[(kElement ? min(e, count - 1) : e) * a.table_lanes];
              const float x = fu[e], y = fv[e];
              fu[e] = x * m.x - y * m.y;
              fv[e] = x * m.z + y * m.w;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float* f = e < 2 ? fu : fv;
              const float4 m = t[e * a.table_lanes];
              const float x = f[2 * (e & 1)], y = f[2 * (e & 1) + 1];
              f[2 * (e & 1)] = x * m.x;
              f[2 * (e & 1) + 1] = y * m.w;
              if (!kElement || e < left) {
                f[2 * (e & 1)] = fmaf(-y, m.y, f[2 * (e & 1)]);
                f[2 * (e & 1) + 1] = fmaf(x, m.z, f[2 * (e & 1) + 1]);
              }
            }
          }
        } else {
          const float2* t = plain + entry;
          if (kHalf) {
#pragma unroll
            for (int e = 0; e < C; ++e) {
              const float2 m = t[(kElement ? min(e, count - 1) : e) * a.table_lanes];
              const float x = fu[e], y = fv[e];
              fu[e] = x * m.x - y * m.y;
              fv[e] = x * m.y + y * m.x;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float* f = e < 2 ? fu : fv;
              const float2 m = t[e * a.table_lanes];
              const float x = f[2 * (e & 1)], y = f[2 * (e & 1) + 1];
              f[2 * (e & 1)] = x * m.x;
              f[2 * (e & 1) + 1] = y * m.x;
              if (!kElement || e < left) {
                f[2 * (e & 1)] = fmaf(-y, m.y, f[2 * (e & 1)]);
                f[2 * (e & 1) + 1] = fmaf(x, m.y, f[2 * (e & 1) + 1]);
              }
            }
          }
        }
      }
      T* to = (it.is_q ? q_to + it.token * a.q_to[1] + static_cast<int64_t>(it.head) * a.q_to_head
                       : k_to + it.token * a.k_to[1] + static_cast<int64_t>(it.head) * a.k_to_head) + first;
      const Chunk<C> ru = narrow<C>(fu, tag), rv = narrow<C>(fv, tag);
      if (!kHalf) {
        *reinterpret_cast<uint4*>(to) = make_uint4(ru.w[0], ru.w[C / 2 - 1], rv.w[0], rv.w[C / 2 - 1]);
      } else if (kElement) {
        store_elements<C>(to, ru, count);
        store_elements<C>(to + apart, rv, count2);
      } else {
        store_chunk<C>(to, ru);
        if (on2) store_chunk<C>(to + apart, rv);
      }
    }
  }
}

template <typename T, bool kHalf, int C, bool kElement, int kNorm>
int launch_mode(RotaryArgs a, int64_t batch, cudaStream_t stream) {
  const int all_heads = a.heads + a.kv_heads;
  a.chunks = kHalf ? (a.pairs + C - 1) / C + (a.dim - 2 * a.pairs + 2 * C - 1) / (2 * C) : a.dim / 8;
  a.lanes_log2 = 0;
  while ((1 << a.lanes_log2) < a.chunks) ++a.lanes_log2;
  a.table_rows = kHalf ? C : 4;
  a.table_lanes = kHalf ? (a.pairs + C - 1) / C : a.dim / 8;
  auto magic = [](int d) { return d == 1 ? 0u : static_cast<uint32_t>(((uint64_t{1} << 32) + d - 1) / d); };
  a.heads_magic = magic(all_heads);
  a.token_magic = magic(a.table_rows * a.table_lanes);
  a.row_magic = magic(a.table_lanes);
  // tokens of a block: angles for all its threads, but no fewer blocks than a few per SM; the norm over a token's heads
  // takes as many as its threads hold at one time
  const int64_t tokens = a.length * batch;
  int per_block = 512 / a.dim > 0 ? 512 / a.dim : 1;
  constexpr int kFewBlocks = 4 * 148;  // four for each SM
  while (per_block > 1 && tokens / per_block < kFewBlocks) --per_block;
  if (kNorm == SQ_ROTARY_NORM_TOKEN)
    while (per_block > 1 && per_block * all_heads > 4 * (256 >> a.lanes_log2)) --per_block;
  a.tokens_per_block = per_block;
  const size_t entries = static_cast<size_t>(per_block) * a.table_rows * a.table_lanes;
  size_t smem = kNorm == SQ_ROTARY_NORM_HEAD ? 32 * entries : 8 * entries;
  if (kNorm == SQ_ROTARY_NORM_TOKEN) smem += sizeof(float) * static_cast<size_t>(per_block) * (all_heads + 2);
  const int64_t per_batch = (a.length + per_block - 1) / per_block;
  if (per_batch > 0x7FFFFFFF / batch) return SQ_ERR_SHAPE;
  a.blocks_per_batch = static_cast<uint32_t>(per_batch);
  sq_rotary_kernel<T, kHalf, C, kElement, kNorm><<<static_cast<unsigned>(per_batch * batch), 256, smem, stream>>>(a);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? SQ_OK : static_cast<int>(err);
}

template <typename T, bool kHalf, int C, bool kElement>
int launch_norm(const RotaryArgs& a, int64_t batch, int norm, cudaStream_t stream) {
  if (norm == SQ_ROTARY_NORM_HEAD) return launch_mode<T, kHalf, C, kElement, SQ_ROTARY_NORM_HEAD>(a, batch, stream);
  if (norm == SQ_ROTARY_NORM_TOKEN) return launch_mode<T, kHalf, C, kElement, SQ_ROTARY_NORM_TOKEN>(a, batch, stream);
  return launch_mode<T, kHalf, C, kElement, SQ_ROTARY_NORM_NONE>(a, batch, stream);
}

// At most 32 chunks in every form (dim <= 256), so a head fits a warp.
template <typename T>
int launch_typed(const RotaryArgs& a, int64_t batch, int layout, int norm, cudaStream_t stream) {
  if (layout == SQ_ROTARY_INTERLEAVED)
    return 2 * a.pairs == a.dim ? launch_norm<T, false, 4, false>(a, batch, norm, stream) : launch_norm<T, false, 4, true>(a, batch, norm, stream);
  if (a.pairs % 8 == 0) return launch_norm<T, true, 8, false>(a, batch, norm, stream);
  if (a.pairs % 4 == 0) return launch_norm<T, true, 4, false>(a, batch, norm, stream);
  return launch_norm<T, true, 8, true>(a, batch, norm, stream);
}

}  // namespace

// q_out may be q and k_out may be k, index by index; else what is written shares memory with nothing.
static int rotary_overlap(const SqRotary& r, int pairs) {
  auto heads = [&](const void* at, int32_t count, const int64_t (&s)[3]) {
    return View(at, 2 * r.dim, r.batch, 2 * s[0], r.length, 2 * s[1], count, 2 * s[2]);
  };
  const int weights = r.norm == SQ_ROTARY_NORM_TOKEN ? r.dim : 0, size = r.position_type == SQ_POS_INT64 ? 8 : 4;
  const View out[2] = {heads(r.q_out, r.heads, r.q_out_strides), heads(r.k_out, r.kv_heads, r.k_out_strides)};
  const View read[6] = {heads(r.q, r.heads, r.q_strides),
                        heads(r.k, r.kv_heads, r.k_strides),
                        View(r.q_weight, (r.q_weight_fp32 ? 4 : 2) * (weights > 0 ? weights * r.heads : r.dim)),
                        View(r.k_weight, (r.k_weight_fp32 ? 4 : 2) * (weights > 0 ? weights * r.kv_heads : r.dim)),
                        View(r.positions, size * r.axes, r.batch, size * r.position_batch_stride, r.length, size * r.position_token_stride),
                        View(r.inv_freq, 8 * pairs)};
  for (int i = 0; i < 2; ++i) {
    if (overlaps_itself(out[i])) return SQ_ERR_OVERLAP;
    for (int j = 0; j < 6; ++j)
      if (overlaps(out[i], read[j]) && !(i == j && same_view(out[i], read[j]))) return SQ_ERR_OVERLAP;
  }
  return overlaps(out[0], out[1]) ? SQ_ERR_OVERLAP : SQ_OK;
}

int launch_rotary(const SqRotary& r, cudaStream_t stream) {
  if (r.q == nullptr || r.q_out == nullptr || r.positions == nullptr || r.inv_freq == nullptr) return SQ_ERR_NULL;
  if (r.kv_heads > 0 && (r.k == nullptr || r.k_out == nullptr)) return SQ_ERR_NULL;
  if (r.dtype != SQ_BF16 && r.dtype != SQ_FP16) return SQ_ERR_ENUM;
  if (r.layout != SQ_ROTARY_INTERLEAVED && r.layout != SQ_ROTARY_HALF) return SQ_ERR_ENUM;
  if (r.norm != SQ_ROTARY_NORM_NONE && r.norm != SQ_ROTARY_NORM_HEAD && r.norm != SQ_ROTARY_NORM_TOKEN) return SQ_ERR_ENUM;
  if (r.position_type != SQ_POS_INT32 && r.position_type != SQ_POS_INT64 && r.position_type != SQ_POS_FP32) return SQ_ERR_ENUM;
  if (r.norm == SQ_ROTARY_NORM_NONE && (r.q_weight != nullptr || r.k_weight != nullptr)) return SQ_ERR_ENUM;
  if (r.batch < 0 || r.length < 0 || r.heads <= 0 || r.kv_heads < 0 || r.dim <= 0 || r.dim % 8 != 0 || r.dim > 256)
    return SQ_ERR_SHAPE;
  if (r.axes < 1 || r.axes > SQ_ROTARY_AXES) return SQ_ERR_SHAPE;
  RotaryArgs a = {};
  int end = 0;
  for (int x = 0; x < SQ_ROTARY_AXES; ++x) {
    if (x < r.axes) {
      if (r.sections[x] < 0 || r.sections[x] > 128) return SQ_ERR_SHAPE;
      end += r.sections[x];
    }
    a.section_end[x] = end;
  }
  if (end < 1 || 2 * end > r.dim) return SQ_ERR_SHAPE;
  int64_t lanes = 1;
  while (8 * lanes < r.dim) lanes *= 2;
  if ((static_cast<int64_t>(r.heads) + r.kv_heads) * lanes > 4096) return SQ_ERR_SHAPE;  // items of a block stay below 2^20
  for (const void* p : {r.q, r.k, static_cast<const void*>(r.q_out), static_cast<const void*>(r.k_out)})
    if (!aligned16_host(p)) return SQ_ERR_SHAPE;
  if (!aligned_param_host(r.q_weight, r.q_weight_fp32 != 0) || !aligned_param_host(r.k_weight, r.k_weight_fp32 != 0)) return SQ_ERR_SHAPE;
  for (const int64_t* s : {r.q_strides, r.k_strides, r.q_out_strides, r.k_out_strides})
    for (int i = 0; i < 3; ++i) {
      if ((s == r.k_strides || s == r.k_out_strides) && r.kv_heads == 0) continue;
      if (s[i] < 0 || s[i] % 8 != 0) return SQ_ERR_SHAPE;  // every vector of every head stays 16-byte aligned
    }
  const uintptr_t position_align = r.position_type == SQ_POS_INT64 ? 7u : 3u;
  if ((reinterpret_cast<uintptr_t>(r.positions) & position_align) != 0) return SQ_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(r.inv_freq) & 7u) != 0) return SQ_ERR_SHAPE;
  if (r.batch > 0 && r.length > (int64_t{1} << 40) / r.batch) return SQ_ERR_SHAPE;
  if (r.batch * r.length == 0) return SQ_OK;
  const int overlap = rotary_overlap(r, end);
  if (overlap != SQ_OK) return overlap;
  a.q = r.q;
  a.k = r.k;
  a.q_out = r.q_out;
  a.k_out = r.k_out;
  for (int i = 0; i < 2; ++i) {
    a.q_in[i] = r.q_strides[i];
    a.k_in[i] = r.k_strides[i];
    a.q_to[i] = r.q_out_strides[i];
    a.k_to[i] = r.k_out_strides[i];
  }
  const int64_t far = 0x7FFFFFFF;  // a head's stride is kept in 32 bits (its multiples are not)
  if (r.q_strides[2] > far || r.q_out_strides[2] > far || (r.kv_heads > 0 && (r.k_strides[2] > far || r.k_out_strides[2] > far)))
    return SQ_ERR_SHAPE;
  a.q_in_head = static_cast<int>(r.q_strides[2]);
  a.q_to_head = static_cast<int>(r.q_out_strides[2]);
  if (r.kv_heads > 0) {
    a.k_in_head = static_cast<int>(r.k_strides[2]);
    a.k_to_head = static_cast<int>(r.k_out_strides[2]);
  }
  a.q_weight = r.q_weight;
  a.k_weight = r.k_weight;
  a.q_weight_f32 = r.q_weight_fp32;
  a.k_weight_f32 = r.k_weight_fp32;
  a.positions = r.positions;
  a.position_type = r.position_type;
  a.position_batch = r.position_batch_stride;
  a.position_token = r.position_token_stride;
  a.inv_freq = r.inv_freq;
  a.length = r.length;
  a.heads = r.heads;
  a.kv_heads = r.kv_heads;
  a.dim = r.dim;
  a.pairs = end;
  a.eps = r.eps;
  a.inv_dim = 1.0f / static_cast<float>(r.dim);
  // batches that lie behind one another like more tokens of one batch are that: short batches share blocks
  int64_t batch = r.batch;
  auto behind = [&](const int64_t (&s)[2]) { return s[0] == r.length * s[1]; };
  if (behind(a.q_in) && behind(a.q_to) && (r.kv_heads == 0 || (behind(a.k_in) && behind(a.k_to))) &&
      a.position_batch == r.length * a.position_token) {
    a.length *= batch;
    batch = 1;
  }
  return r.dtype == SQ_BF16 ? launch_typed<__nv_bfloat16>(a, batch, r.layout, r.norm, stream)
                            : launch_typed<__half>(a, batch, r.layout, r.norm, stream);
}

}  // namespace sq
