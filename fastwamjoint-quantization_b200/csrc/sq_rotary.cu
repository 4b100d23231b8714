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
// A head is covered by `lanes` lanes (the power of two that holds dim / 8 vectors), a block by whole tokens.  A lane
// loads all its vectors before the angles are computed.  Per-head sums are shuffles inside the lanes of a head; the
// norm over a token's heads adds those sums in head order through shared memory.
#include "sq_internal.h"
#include "sq_rows.cuh"

namespace sq {
namespace {

constexpr int kInterleaved = 0, kHalfVector = 1, kHalfElement = 2;  // how a lane reaches the other element of a pair

struct RotaryArgs {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int64_t q_in[3], k_in[3], q_to[3], k_to[3];  // strides in elements: batch, token, head
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
  int lanes_log2, tokens_per_block;
  float eps;
};

__device__ __forceinline__ double position_at(const RotaryArgs& a, int64_t at) {
  if (a.position_type == SQ_POS_INT32) return static_cast<double>(static_cast<const int32_t*>(a.positions)[at]);
  if (a.position_type == SQ_POS_INT64) return static_cast<double>(static_cast<const int64_t*>(a.positions)[at]);
  return static_cast<double>(static_cast<const float*>(a.positions)[at]);
}

template <typename T, int kMode, int kNorm, int VPT>
__global__ void __launch_bounds__(256) sq_rotary_kernel(const RotaryArgs a) {
  extern __shared__ __align__(16) float smem[];
  const T* tag = nullptr;
  const int half = a.dim / 2;                         // angle slots of a token; those past `pairs` hold the identity
  float2* turn = reinterpret_cast<float2*>(smem);     // [tokens_per_block][half]
  float* sums = smem + 2 * a.tokens_per_block * half; // token norm: [tokens_per_block][heads + kv_heads], then 1 / rms
  float* stage = sums + (kNorm == SQ_ROTARY_NORM_TOKEN ? a.tokens_per_block * (a.heads + a.kv_heads + 2) : 0);

  const int lanes = 1 << a.lanes_log2;
  const int v = threadIdx.x & (lanes - 1);            // vector of the head
  const int all_heads = a.heads + a.kv_heads;
  const uint32_t batch = blockIdx.x / a.blocks_per_batch;
  const int64_t first_token = static_cast<int64_t>(blockIdx.x - batch * a.blocks_per_batch) * a.tokens_per_block;
  const int here = static_cast<int>(min(static_cast<int64_t>(a.tokens_per_block), a.length - first_token));
  const T* q = static_cast<const T*>(a.q) + batch * a.q_in[0] + first_token * a.q_in[1];
  const T* k = static_cast<const T*>(a.k) + batch * a.k_in[0] + first_token * a.k_in[1];
  const int segments = blockDim.x >> a.lanes_log2;    // heads a block takes at a time

  uint4 raw[VPT];
  bool on[VPT];
  int local[VPT], head[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int item = i * segments + static_cast<int>(threadIdx.x >> a.lanes_log2);
    local[i] = item / all_heads;
    head[i] = item - local[i] * all_heads;
    on[i] = local[i] < here && v * 8 < a.dim;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (on[i]) {
      const bool is_q = head[i] < a.heads;
      raw[i] = load_stream((is_q ? q + local[i] * a.q_in[1] + head[i] * a.q_in[2]
                                 : k + local[i] * a.k_in[1] + (head[i] - a.heads) * a.k_in[2]) + v * 8);
    }
  }
  for (int i = threadIdx.x; i < here * half; i += blockDim.x) {
    const int token_here = i / half, j = i - token_here * half;
    float2 cs = make_float2(1.0f, 0.0f);
    if (j < a.pairs) {
      int axis = 0;
#pragma unroll
      for (int x = 0; x < SQ_ROTARY_AXES - 1; ++x) axis += j >= a.section_end[x] ? 1 : 0;
      const int64_t at = batch * a.position_batch + (first_token + token_here) * a.position_token + axis;
      const double turns = position_at(a, at) * a.inv_freq[j] * 0.15915494309189533577;  // 1 / (2 pi)
      const float part = static_cast<float>(turns - rint(turns));
      sincospif(2.0f * part, &cs.y, &cs.x);
    }
    turn[i] = cs;
  }
  __syncthreads();

  float scale[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) scale[i] = 1.0f;
  if (kNorm != SQ_ROTARY_NORM_NONE) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float f[8];
      unpack8(raw[i], f, tag);
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(f[e], f[e], s);
      for (int d = lanes >> 1; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (kNorm == SQ_ROTARY_NORM_HEAD) scale[i] = rsqrtf(s / static_cast<float>(a.dim) + a.eps);
      else if (v == 0 && local[i] < here) sums[local[i] * all_heads + head[i]] = s;
    }
  }
  if (kNorm == SQ_ROTARY_NORM_TOKEN) {
    __syncthreads();
    float* roots = sums + a.tokens_per_block * all_heads;  // [tokens_per_block][q, k]
    for (int i = threadIdx.x >> 5; i < 2 * here; i += blockDim.x >> 5) {  // a warp per (token, q or k)
      const int begin = (i & 1) ? a.heads : 0, count = (i & 1) ? a.kv_heads : a.heads;
      float s = 0.0f;
      for (int hd = threadIdx.x & 31; hd < count; hd += 32) s += sums[(i >> 1) * all_heads + begin + hd];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if ((threadIdx.x & 31) == 0) roots[i] = rsqrtf(s / (static_cast<float>(count) * static_cast<float>(a.dim)) + a.eps);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (local[i] < here) scale[i] = roots[2 * local[i] + (head[i] < a.heads ? 0 : 1)];
  }

#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float f[8], out[8];
    unpack8(raw[i], f, tag);
    const bool is_q = head[i] < a.heads;
    const int own_head = is_q ? head[i] : head[i] - a.heads;
    if (kNorm != SQ_ROTARY_NORM_NONE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= scale[i];
      const void* w = is_q ? a.q_weight : a.k_weight;
      if (w != nullptr && on[i]) {
        float p[8];
        const int64_t at = (kNorm == SQ_ROTARY_NORM_TOKEN ? own_head * a.dim : 0) + v * 8;
        load_params<T>(w, at, (is_q ? a.q_weight_f32 : a.k_weight_f32) != 0, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= p[e];
      }
    }
    const float2* angles = turn + (on[i] ? local[i] * half : 0);
    if (kMode == kInterleaved) {
      if (on[i]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 cs = angles[v * 4 + j];
          out[2 * j] = f[2 * j] * cs.x - f[2 * j + 1] * cs.y;
          out[2 * j + 1] = f[2 * j] * cs.y + f[2 * j + 1] * cs.x;
        }
      }
    } else if (kMode == kHalfVector) {
      // pairs % 8 == 0: the partners of a vector are one vector, in another lane of the head
      const int step = a.pairs / 8;
      const int other = v < step ? v + step : v < 2 * step ? v - step : v;
      const int source = (static_cast<int>(threadIdx.x & 31) & ~(lanes - 1)) | other;
      const int j0 = v < step ? v * 8 : (v - step) * 8;
      const float sign = v < step ? -1.0f : 1.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float partner = __shfl_sync(0xffffffffu, f[e], source);
        if (v < 2 * step) {
          const float2 cs = angles[j0 + e];
          out[e] = f[e] * cs.x + sign * partner * cs.y;
        } else {
          out[e] = f[e];
        }
      }
    } else {
      // pairs of any number: the head goes through shared memory, partners are picked element by element
      float* mine = stage + (threadIdx.x >> a.lanes_log2) * a.dim;
      __syncwarp();  // the last head's readers are done
      if (on[i]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) mine[v * 8 + e] = f[e];
      }
      __syncwarp();
      if (on[i]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int x = v * 8 + e;
          if (x < a.pairs) {
            const float2 cs = angles[x];
            out[e] = f[e] * cs.x - mine[x + a.pairs] * cs.y;
          } else if (x < 2 * a.pairs) {
            const float2 cs = angles[x - a.pairs];
            out[e] = f[e] * cs.x + mine[x - a.pairs] * cs.y;
          } else {
            out[e] = f[e];
          }
        }
      }
    }
    if (on[i]) {
      const int64_t t = first_token + local[i];
      T* to = is_q ? static_cast<T*>(a.q_out) + batch * a.q_to[0] + t * a.q_to[1] + own_head * a.q_to[2]
                   : static_cast<T*>(a.k_out) + batch * a.k_to[0] + t * a.k_to[1] + own_head * a.k_to[2];
      *reinterpret_cast<uint4*>(to + v * 8) = pack8(out, tag);
    }
  }
}

template <typename T, int kMode, int kNorm>
int launch_mode(RotaryArgs a, int64_t batch, cudaStream_t stream) {
  const int all_heads = a.heads + a.kv_heads;
  constexpr int kThreads = 256;
  const int segments = kThreads >> a.lanes_log2;
  // whole tokens per block: as many as keep every lane busy once, one where a token's heads need several turns
  a.tokens_per_block = all_heads >= segments ? 1 : segments / all_heads;
  const int turns = (a.tokens_per_block * all_heads + segments - 1) / segments;
  size_t smem = sizeof(float) * 2 * static_cast<size_t>(a.tokens_per_block) * (a.dim / 2);
  if (kNorm == SQ_ROTARY_NORM_TOKEN) smem += sizeof(float) * static_cast<size_t>(a.tokens_per_block) * (all_heads + 2);
  if (kMode == kHalfElement) smem += sizeof(float) * static_cast<size_t>(segments) * a.dim;
  const int64_t per_batch = (a.length + a.tokens_per_block - 1) / a.tokens_per_block;
  if (per_batch > 0x7FFFFFFF / batch || turns > 16) return SQ_ERR_SHAPE;
  a.blocks_per_batch = static_cast<uint32_t>(per_batch);
  const unsigned grid = static_cast<unsigned>(per_batch * batch);
  if (turns <= 1) sq_rotary_kernel<T, kMode, kNorm, 1><<<grid, kThreads, smem, stream>>>(a);
  else if (turns <= 2) sq_rotary_kernel<T, kMode, kNorm, 2><<<grid, kThreads, smem, stream>>>(a);
  else if (turns <= 4) sq_rotary_kernel<T, kMode, kNorm, 4><<<grid, kThreads, smem, stream>>>(a);
  else if (turns <= 8) sq_rotary_kernel<T, kMode, kNorm, 8><<<grid, kThreads, smem, stream>>>(a);
  else sq_rotary_kernel<T, kMode, kNorm, 16><<<grid, kThreads, smem, stream>>>(a);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? SQ_OK : static_cast<int>(err);
}

template <typename T, int kMode>
int launch_norm(const RotaryArgs& a, int64_t batch, int norm, cudaStream_t stream) {
  if (norm == SQ_ROTARY_NORM_HEAD) return launch_mode<T, kMode, SQ_ROTARY_NORM_HEAD>(a, batch, stream);
  if (norm == SQ_ROTARY_NORM_TOKEN) return launch_mode<T, kMode, SQ_ROTARY_NORM_TOKEN>(a, batch, stream);
  return launch_mode<T, kMode, SQ_ROTARY_NORM_NONE>(a, batch, stream);
}

template <typename T>
int launch_typed(const RotaryArgs& a, int64_t batch, int layout, int norm, cudaStream_t stream) {
  if (layout == SQ_ROTARY_INTERLEAVED) return launch_norm<T, kInterleaved>(a, batch, norm, stream);
  if (a.pairs % 8 == 0) return launch_norm<T, kHalfVector>(a, batch, norm, stream);
  return launch_norm<T, kHalfElement>(a, batch, norm, stream);
}

}  // namespace

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
  for (const void* p : {r.q, r.k, static_cast<const void*>(r.q_out), static_cast<const void*>(r.k_out), r.q_weight, r.k_weight})
    if (!aligned16_host(p)) return SQ_ERR_SHAPE;
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
  a.q = r.q;
  a.k = r.k;
  a.q_out = r.q_out;
  a.k_out = r.k_out;
  for (int i = 0; i < 3; ++i) {
    a.q_in[i] = r.q_strides[i];
    a.k_in[i] = r.k_strides[i];
    a.q_to[i] = r.q_out_strides[i];
    a.k_to[i] = r.k_out_strides[i];
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
  while ((8 << a.lanes_log2) < r.dim) ++a.lanes_log2;
  a.eps = r.eps;
  // batches that lie behind one another like more tokens of one batch are that: short batches share blocks
  int64_t batch = r.batch;
  auto behind = [&](const int64_t (&s)[3]) { return s[0] == r.length * s[1]; };
  if (behind(a.q_in) && behind(a.q_to) && (r.kv_heads == 0 || (behind(a.k_in) && behind(a.k_to))) &&
      a.position_batch == r.length * a.position_token) {
    a.length *= batch;
    batch = 1;
  }
  return r.dtype == SQ_BF16 ? launch_typed<__nv_bfloat16>(a, batch, r.layout, r.norm, stream)
                            : launch_typed<__half>(a, batch, r.layout, r.norm, stream);
}

}  // namespace sq
