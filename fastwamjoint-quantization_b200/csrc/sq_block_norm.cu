// Norms before and after a block with its gate and residual scale, and the e4m3 quantizer.
//
//   b = post(branch) * post_weight + post_bias
//   h = residual_scale * x + gate * b                       written in the rows' type
//   z = (norm(h) * weight + bias) * (1 + scale) + shift     written in the rows' type, or as e4m3 codes and scales
//
// with post / norm the RMS or layer norm of a row, statistics and all arithmetic in fp32 from the unrounded h (one
// rounding per output).  A row lives in registers between its loads and its stores, so each element is read once and
// written once: the kernel is bound by HBM.  The layer norm takes its variance from the deviations (a second reduction
// in registers), not from the difference of two sums.
#include <type_traits>

#include "sq_internal.h"
#include "sq_overlap.h"
#include "sq_rows.cuh"

namespace sq {
namespace {

// Rows of [width], `stride` elements apart, one for each `span` rows of x: row / span is the high word of row * magic
// shifted right (magic 0: span 1, or one row for all and stride 0).  Three divisions per thread were 45 of its 300 instructions.
struct Param {
  const void* p;
  int64_t stride;
  uint32_t magic, shift;
  int f32;
};

struct NormArgs {
  const void* x;
  const void* branch;
  Param gate, post_weight, post_bias, weight, bias, mod_scale, mod_shift;
  float residual_scale, eps, inv_width;
  int post_kind, norm_kind;
  void* h_out;
  void* z_out;
  float* scales;
  int64_t scales_row, scales_group;
  int64_t rows;
  int width;
};

// Sum over the threads of a block, the same value in each of them and the same order in every run.  Two buffers in turn:
// one barrier per sum (a buffer is written again two sums later, past the barrier of the sum between).  Up to eight warps'
// parts are added by every thread: two wide reads of the same address and a short tree take less time than shuffles
// (measured with the divisions below: 32768 x 4096 at 221 us where it took 231); sixteen and more parts cost registers that spill.
template <int kWarps>
struct RowSum {
  static constexpr int kParts = kWarps < 4 ? 4 : kWarps;
  float* partial;  // [2][kParts]
  int buffer = 0;
  __device__ __forceinline__ explicit RowSum(float* memory) : partial(memory) {
    // parts of warps that this width does not have; the barrier of the first sum orders them
    if (threadIdx.x < 2 * kParts && (threadIdx.x & (kParts - 1)) >= (blockDim.x >> 5)) partial[threadIdx.x] = 0.0f;
  }
  __device__ __forceinline__ float operator()(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    float* mine = partial + buffer * kParts;
    buffer ^= 1;
    if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = v;
    __syncthreads();
    if constexpr (kParts > 8) {
      v = mine[threadIdx.x & (kParts - 1)];
#pragma unroll
      for (int d = kParts / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
      return v;
    }
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < kParts; i += 4) {
      const float4 q = *reinterpret_cast<const float4*>(mine + i);
      total += (q.x + q.y) + (q.z + q.w);
    }
    return total;
  }
};

template <int VPT>
__device__ __forceinline__ float local_squares(const float (&v)[VPT][8]) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(v[i][e], v[i][e], s);
  }
  return s;
}

// v -> (v - mean) / sqrt(variance + eps) or v / sqrt(mean square + eps); slots without elements stay zero
template <int VPT, typename Sum>
__device__ __forceinline__ void standardise(float (&v)[VPT][8], const bool (&on)[VPT], int kind, float eps, float inv_width,
                                            Sum& row_sum) {
  if (kind == SQ_NORM_LAYER) {
    float share = 0.0f;  // of the mean: added up as v / width, which cannot overflow
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) share = fmaf(v[i][e], inv_width, share);
    }
    const float mean = row_sum(share);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const float less = on[i] ? mean : 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] -= less;
    }
  }
  float squares = row_sum(local_squares(v));
  float mean_square = fmaf(squares, inv_width, eps);
  if (!(mean_square > 1e-30f && squares < __int_as_float(0x7F800000))) {
    // the squares of bf16 values beyond 2^59 or so overflow, and those of tiny ones vanish where eps does not cover them: the
    // row over again, 2^70 times smaller or larger.  The sum is the same in every thread of the row, so all of them come here
    // or none.
    const float by = squares < 1.0f ? 1180591620717411303424.0f : 8.470329472543003e-22f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] *= by;
    }
    squares = row_sum(local_squares(v));
    mean_square = fmaf(squares, inv_width, eps * by * by);
  }
  const float r = __frsqrt_rn(mean_square);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] *= r;
  }
}

// where a row's parameters start
__device__ __forceinline__ int64_t param_base(const Param& q, uint32_t row) {
  return static_cast<int64_t>(q.magic != 0 ? __umulhi(row, q.magic) >> q.shift : row) * q.stride;
}

// A block takes a row, thread t owning the vectors t and t + blockDim: a warp reads 512 contiguous bytes, and the 16 vectors
// of a run of 128 sit in 16 neighbouring lanes.
template <typename T, int VPT, bool kBranch, int kMaxThreads, int kMinBlocks>
__global__ void __launch_bounds__(kMaxThreads, kMinBlocks) sq_block_norm_kernel(const NormArgs a) {
  __shared__ __align__(16) float partial[2 * RowSum<kMaxThreads / 32>::kParts];
  RowSum<kMaxThreads / 32> row_sum(partial);
  const T* tag = nullptr;
  const uint32_t row = blockIdx.x;
  const int64_t base = static_cast<int64_t>(row) * a.width;
  int column[VPT];
  bool on[VPT];
  uint4 raw_x[VPT], raw_b[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    column[i] = static_cast<int>(threadIdx.x + i * blockDim.x) * 8;
    on[i] = column[i] < a.width;
    raw_x[i] = on[i] ? load_stream(static_cast<const T*>(a.x) + base + column[i]) : make_uint4(0, 0, 0, 0);
    if (kBranch) raw_b[i] = on[i] ? load_stream(static_cast<const T*>(a.branch) + base + column[i]) : make_uint4(0, 0, 0, 0);
  }
  const int64_t gate_base = kBranch ? param_base(a.gate, row) : 0;
  const int64_t scale_base = param_base(a.mod_scale, row), shift_base = param_base(a.mod_shift, row);
  float h[VPT][8], p[8];
  if (kBranch) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) unpack8(raw_b[i], h[i], tag);
    if (a.post_kind != SQ_NORM_NONE) {
      standardise<VPT>(h, on, a.post_kind, a.eps, a.inv_width, row_sum);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (!on[i]) continue;
        if (a.post_weight.p != nullptr) {
          load_params<T>(a.post_weight.p, column[i], a.post_weight.f32 != 0, p);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[i][e] *= p[e];
        }
        if (a.post_bias.p != nullptr) {
          load_params<T>(a.post_bias.p, column[i], a.post_bias.f32 != 0, p);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[i][e] += p[e];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (!on[i]) continue;
      if (a.gate.p != nullptr) {
        load_params<T>(a.gate.p, gate_base + column[i], a.gate.f32 != 0, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] *= p[e];
      }
      float xv[8];
      unpack8(raw_x[i], xv, tag);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] = fmaf(a.residual_scale, xv[e], h[i][e]);
      *reinterpret_cast<uint4*>(static_cast<T*>(a.h_out) + base + column[i]) = pack8(h[i], tag);
    }
    if (a.norm_kind == SQ_NORM_NONE) return;
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) unpack8(raw_x[i], h[i], tag);
  }
  standardise<VPT>(h, on, a.norm_kind, a.eps, a.inv_width, row_sum);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (on[i]) {
      if (a.weight.p != nullptr) {
        load_params<T>(a.weight.p, column[i], a.weight.f32 != 0, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] *= p[e];
      }
      if (a.bias.p != nullptr) {
        load_params<T>(a.bias.p, column[i], a.bias.f32 != 0, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] += p[e];
      }
      if (a.mod_scale.p != nullptr) {
        load_params<T>(a.mod_scale.p, scale_base + column[i], a.mod_scale.f32 != 0, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] = fmaf(h[i][e], p[e], h[i][e]);
      }
      if (a.mod_shift.p != nullptr) {
        load_params<T>(a.mod_shift.p, shift_base + column[i], a.mod_shift.f32 != 0, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] += p[e];
      }
      if (a.scales == nullptr) *reinterpret_cast<uint4*>(static_cast<T*>(a.z_out) + base + column[i]) = pack8(h[i], tag);
    }
    if (a.scales != nullptr) {  // every lane of the warp is here: the run's maximum is a shuffle
      const float s = e4m3_scale(run_max(on[i] ? magnitude8(h[i]) : 0u));
      if (on[i]) {
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.z_out) + base + column[i]) = quantize8(h[i], __fdiv_rn(1.0f, s));
        if ((threadIdx.x & 15) == 0) a.scales[row * a.scales_row + (column[i] >> 7) * a.scales_group] = s;
      }
    }
  }
}

template <typename T, int VPT, int kMaxThreads, int kMinBlocks>
int launch_shape(const NormArgs& a, cudaStream_t stream) {
  const int threads = (a.width / 8 + VPT * 32 - 1) / (VPT * 32) * 32;
  const unsigned blocks = static_cast<unsigned>(a.rows);
  if (a.branch != nullptr) sq_block_norm_kernel<T, VPT, true, kMaxThreads, kMinBlocks><<<blocks, threads, 0, stream>>>(a);
  else sq_block_norm_kernel<T, VPT, false, kMaxThreads, kMinBlocks><<<blocks, threads, 0, stream>>>(a);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? SQ_OK : static_cast<int>(err);
}

// One vector per thread up to 1024 elements, else two; registers are held to what lets 64 / 48 warps live on an SM: the more
// rows under way, the better HBM is used.  The forms with a branch pay for it with spills (ptxas: 16 to 64 bytes of stores a
// thread beyond 1024 elements), and are faster all the same.  Measured at 32768 x 4096 fp16 with fp32 modulation, before its
// parameters were read 32 bytes at a time: two vectors and 32 / 40 / 48 / 64 warps 259 / 233 / 236 / 289 us, one vector and 64
// warps 247 (225 now); at 4096 x 5120 with a modulation row per token 72 / 72 / 61 / 62 us; at 32 x 1024 one vector 2.4 us,
// two 3.2.  Beyond 8192 a block of two vectors per thread fills an SM, and two blocks of four vectors overlap one's loads with
// the other's sums.  With two rows for each of 148 SMs or more that is faster on the whole; two RMS norms, two vectors against
// four: 12288 wide 9.6 / 9.8 us at 296 rows, 13.4 / 15.9 at 444, 18.4 / 18.0 at 592, 228 / 193 at 8192; 16384 wide 11.6 / 10.8,
// 17.5 / 19.7, 25 / 23.8, 280 / 245.  Where 64 rows leave SMs idle it is 8.2 instead of 5.7.
template <typename T>
int launch_typed(const NormArgs& a, cudaStream_t stream) {
  if (a.width <= 512) return launch_shape<T, 1, 64, 32>(a, stream);
  if (a.width <= 1024) return launch_shape<T, 1, 128, 16>(a, stream);
  if (a.width <= 2048) return launch_shape<T, 2, 128, 12>(a, stream);
  if (a.width <= 4096) return launch_shape<T, 2, 256, 6>(a, stream);
  if (a.width <= 8192) return launch_shape<T, 2, 512, 3>(a, stream);
  if (a.rows >= 2 * 148) return launch_shape<T, 4, 512, 2>(a, stream);
  return launch_shape<T, 2, 1024, 1>(a, stream);
}

// ---------------------------------------------------------------------------------------------- e4m3 quantizer
// 16 lanes per run of 128, kRuns runs per thread loaded before the first is used.  No row statistics are needed, so runs are
// dealt out regardless of rows; the row of a run is a multiplication by the reciprocal of the runs per row (exact for run
// numbers below 2^31).  Two runs and registers for eight blocks per SM: four runs at five blocks take 2.3 us instead of 1.8
// for one token of 4096, 62.9 instead of 64.4 for 8192 of 14336, and with the activation 114 instead of 109.
constexpr int kRuns = 2;
constexpr int kQuantThreads = 256;

template <typename T, bool kGelu>
__global__ void __launch_bounds__(kQuantThreads, 8) sq_fp8_quantize_kernel(
    const T* __restrict__ x, uint8_t* __restrict__ codes, float* __restrict__ scales, int64_t scales_row,
    int64_t scales_group, uint32_t runs, uint32_t runs_per_row, uint32_t magic, uint32_t shift, int width) {
  // the product behind this kernel may set itself up meanwhile; it waits for this grid before it reads anything of it
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane16 = threadIdx.x & 15;
  const uint32_t first = blockIdx.x * (kQuantThreads / 16 * kRuns) + (threadIdx.x >> 4);
  uint4 raw[kRuns];
  uint32_t row[kRuns], group[kRuns];
  bool on[kRuns];
#pragma unroll
  for (int i = 0; i < kRuns; ++i) {
    const uint32_t run = first + i * (kQuantThreads / 16);
    row[i] = runs_per_row == 1 ? run : __umulhi(run, magic) >> shift;
    group[i] = run - row[i] * runs_per_row;
    const int column = static_cast<int>(group[i]) * 128 + lane16 * 8;
    on[i] = run < runs && column < width;
    raw[i] = on[i] ? load_stream(x + static_cast<int64_t>(row[i]) * width + column) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < kRuns; ++i) {
    float v[8];
    unpack8(raw[i], v, static_cast<const T*>(nullptr));
    if (kGelu) gelu8(v);
    const float s = e4m3_scale(run_max(magnitude8(v)));
    if (on[i]) {
      const int64_t at = static_cast<int64_t>(row[i]) * width + static_cast<int64_t>(group[i]) * 128 + lane16 * 8;
      *reinterpret_cast<uint2*>(codes + at) = quantize8(v, __fdiv_rn(1.0f, s));
      if (lane16 == 0) scales[static_cast<int64_t>(row[i]) * scales_row + static_cast<int64_t>(group[i]) * scales_group] = s;
    }
  }
}

// n / d = (n * magic) >> (32 + shift) with magic = ceil(2^(32 + shift) / d), 2^shift < d <= 2^(shift + 1): the error
// n * (magic * d - 2^(32 + shift)) stays below 2^(32 + shift) for n < 2^31.  d = 1 has no such form: magic 0.
struct Divisor {
  uint32_t magic, shift;
};
Divisor divisor(int64_t d) {
  uint32_t shift = 0;
  while ((int64_t{2} << shift) < d) ++shift;
  return {d == 1 ? 0 : static_cast<uint32_t>(((uint64_t{1} << (32 + shift)) + d - 1) / d), shift};
}

}  // namespace

int launch_fp8_quantize(const void* x, int x_dtype, int64_t rows, int64_t K, int input_activation, void* codes, float* scales,
                        int64_t scales_row, int64_t scales_group, cudaStream_t stream) {
  if (x == nullptr || codes == nullptr || scales == nullptr) return SQ_ERR_NULL;
  if (x_dtype != SQ_BF16 && x_dtype != SQ_FP16) return SQ_ERR_ENUM;
  if (input_activation != SQ_ACT_FN_NONE && input_activation != SQ_ACT_FN_GELU) return SQ_ERR_ENUM;
  if (rows < 0 || K <= 0 || K % 16 != 0 || K > 131072) return SQ_ERR_SHAPE;
  if (!aligned16_host(x) || !aligned16_host(codes) || (reinterpret_cast<uintptr_t>(scales) & 3u) != 0) return SQ_ERR_SHAPE;
  if (rows == 0) return SQ_OK;
  const int64_t per_row = (K + 127) / 128;
  if (rows > (int64_t{1} << 30) / per_row) return SQ_ERR_SHAPE;
  if (scales_row < 0 || scales_group < 0) return SQ_ERR_SHAPE;
  const View from(x, rows * K * 2), to(codes, rows * K), scale_view(scales, 4, per_row, scales_group * 4, rows, scales_row * 4);
  if (clashes(to, {from, scale_view}) || clashes(scale_view, {from})) return SQ_ERR_OVERLAP;
  const uint32_t runs = static_cast<uint32_t>(rows * per_row);
  const Divisor by = divisor(per_row);
  const unsigned blocks = (runs + kQuantThreads / 16 * kRuns - 1) / (kQuantThreads / 16 * kRuns);
  auto go = [&](auto tag, auto gelu) {
    using T = decltype(tag);
    sq_fp8_quantize_kernel<T, decltype(gelu)::value><<<blocks, kQuantThreads, 0, stream>>>(
        static_cast<const T*>(x), static_cast<uint8_t*>(codes), scales, scales_row, scales_group, runs,
        static_cast<uint32_t>(per_row), by.magic, by.shift, static_cast<int>(K));
  };
  const bool gelu = input_activation == SQ_ACT_FN_GELU;
  if (x_dtype == SQ_BF16) gelu ? go(__nv_bfloat16{}, std::true_type{}) : go(__nv_bfloat16{}, std::false_type{});
  else gelu ? go(__half{}, std::true_type{}) : go(__half{}, std::false_type{});
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? SQ_OK : static_cast<int>(err);
}

// h and z may take the place of x or branch, row by row; else what is written shares memory with nothing.
static int norm_overlap(const SqBlockNorm& b) {
  const int64_t bytes = b.rows * b.width;
  const View in[2] = {View(b.x, 2 * bytes), View(b.branch, 2 * bytes)};
  const View out[3] = {View(b.branch != nullptr ? b.h_out : nullptr, 2 * bytes),
                       View(b.norm_kind != SQ_NORM_NONE ? b.z_out : nullptr, b.scales != nullptr ? bytes : 2 * bytes),
                       View(b.scales, 4, (b.width + 127) / 128, 4 * b.scales_group_stride, b.rows, 4 * b.scales_row_stride)};
  const SqParam* params[7] = {&b.gate, &b.mod_scale, &b.mod_shift, &b.post_weight, &b.post_bias, &b.weight, &b.bias};
  for (int i = 0; i < 7; ++i) {
    const SqParam& q = *params[i];
    if (q.data == nullptr) continue;
    const int64_t size = q.is_fp32 ? 4 : 2, rows = i < 3 && q.span < b.rows ? (b.rows + q.span - 1) / q.span : 1;
    const View read(q.data, b.width * size, rows, i < 3 ? q.row_stride * size : 0);
    if (overlaps(out[0], read) || overlaps(out[1], read) || overlaps(out[2], read)) return SQ_ERR_OVERLAP;
  }
  for (int i = 0; i < 3; ++i) {
    if (overlaps_itself(out[i])) return SQ_ERR_OVERLAP;
    for (int j = 0; j < 2; ++j)
      if (overlaps(out[i], in[j]) && !same_view(out[i], in[j])) return SQ_ERR_OVERLAP;
    for (int j = 0; j < i; ++j)
      if (overlaps(out[i], out[j])) return SQ_ERR_OVERLAP;
  }
  return SQ_OK;
}

int launch_block_norm(const SqBlockNorm& b, cudaStream_t stream) {
  if (b.x == nullptr) return SQ_ERR_NULL;
  if (b.dtype != SQ_BF16 && b.dtype != SQ_FP16) return SQ_ERR_ENUM;
  for (const int kind : {b.post_kind, b.norm_kind})
    if (kind != SQ_NORM_NONE && kind != SQ_NORM_LAYER && kind != SQ_NORM_RMS) return SQ_ERR_ENUM;
  if (b.branch == nullptr && b.norm_kind == SQ_NORM_NONE) return SQ_ERR_NULL;
  if ((b.branch != nullptr && b.h_out == nullptr) || (b.norm_kind != SQ_NORM_NONE && b.z_out == nullptr)) return SQ_ERR_NULL;
  if (b.norm_kind == SQ_NORM_NONE && (b.scales != nullptr || b.mod_scale.data != nullptr || b.mod_shift.data != nullptr ||
                                      b.weight.data != nullptr || b.bias.data != nullptr))
    return SQ_ERR_ENUM;  // nothing would read them
  if (b.branch == nullptr && (b.gate.data != nullptr || b.post_kind != SQ_NORM_NONE)) return SQ_ERR_ENUM;
  if (b.post_kind == SQ_NORM_NONE && (b.post_weight.data != nullptr || b.post_bias.data != nullptr)) return SQ_ERR_ENUM;
  if (b.rows < 0 || b.width <= 0 || b.width % (b.scales != nullptr ? 16 : 8) != 0 || b.width > 16384) return SQ_ERR_SHAPE;
  if (b.rows > 0x7FFFFFFF) return SQ_ERR_SHAPE;
  for (const void* p : {b.x, b.branch, static_cast<const void*>(b.h_out), static_cast<const void*>(b.z_out)})
    if (!aligned16_host(p)) return SQ_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(b.scales) & 3u) != 0) return SQ_ERR_SHAPE;
  NormArgs a = {};
  // the per-channel vectors have one row; a span beyond the rows is one row too
  auto row_of = [](const SqParam& q) { return Param{q.data, 0, 0u, 0u, q.is_fp32}; };
  auto take = [&](const SqParam& q) {
    if (q.data == nullptr || q.span >= b.rows) return row_of(q);
    const Divisor by = divisor(q.span);
    return Param{q.data, q.row_stride, by.magic, by.shift, q.is_fp32};
  };
  for (const SqParam* q : {&b.gate, &b.mod_scale, &b.mod_shift})
    if (q->data != nullptr && (q->span <= 0 || q->row_stride < 0 || q->row_stride % 8 != 0)) return SQ_ERR_SHAPE;
  a.gate = take(b.gate);
  a.post_weight = row_of(b.post_weight);
  a.post_bias = row_of(b.post_bias);
  a.weight = row_of(b.weight);
  a.bias = row_of(b.bias);
  a.mod_scale = take(b.mod_scale);
  a.mod_shift = take(b.mod_shift);
  for (const Param& q : {a.gate, a.post_weight, a.post_bias, a.weight, a.bias, a.mod_scale, a.mod_shift})
    if (!aligned_param_host(q.p, q.f32 != 0)) return SQ_ERR_SHAPE;
  if (b.scales != nullptr && (b.scales_row_stride < 0 || b.scales_group_stride < 0)) return SQ_ERR_SHAPE;
  if (b.rows == 0) return SQ_OK;
  const int overlap = norm_overlap(b);
  if (overlap != SQ_OK) return overlap;
  a.x = b.x;
  a.branch = b.branch;
  a.residual_scale = b.residual_scale;
  a.eps = b.eps;
  a.post_kind = b.post_kind;
  a.norm_kind = b.norm_kind;
  a.h_out = b.h_out;
  a.z_out = b.z_out;
  a.scales = b.scales;
  a.scales_row = b.scales_row_stride;
  a.scales_group = b.scales_group_stride;
  a.rows = b.rows;
  a.width = static_cast<int>(b.width);
  a.inv_width = 1.0f / static_cast<float>(b.width);
  return b.dtype == SQ_BF16 ? launch_typed<__nv_bfloat16>(a, stream) : launch_typed<__half>(a, stream);
}

}  // namespace sq
