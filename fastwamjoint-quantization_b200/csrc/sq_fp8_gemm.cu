// 8-bit floating-point matrix product with a scale for each block of 128:
//
//   y[m, n] = sum_g  s[m, g] * t[n / 128, g] * (sum_{k in run g} a[m, k] w[n, k])  + bias[n]
//
// a: e4m3 codes of the tokens with one fp32 scale per token and run of 128 k; w: e4m3 weights with one fp32 scale per
// 128 x 128 block.  The inner sums run on the tensor core (tcgen05.mma kind::f8f6f4, fp32 accumulators in tensor
// memory); since the scales change with every run, each run of 128 k gets an accumulator of its own, which the drain
// warps read back, multiply by the run's scale and add in fp32 registers.
//
// sq_fp8_few_kernel: weights as the rows of the tile (128 output channels = 128 TMEM lanes), tokens as its columns
// (16 .. 128): few tokens make a narrow tile, not an empty one.  When the tiles do not fill the GPU, a cluster of up to 8
// thread blocks splits the K of a tile; the parts meet in distributed shared memory, where each thread block adds
// the parts of its share of the tokens in part order (no atomics: the same result in every run) and stores them in
// 256-byte rows.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <mutex>

#include "sq_internal.h"
#include "sq_ptx.cuh"
#include "sq_rows.cuh"

namespace sq {
namespace {

constexpr uint64_t kWaitLimitNs = 1000000000ull;
constexpr int kRun = 128;  // k of one scale = bytes of one swizzled operand row

struct Fp8Args {
  const float* scales;         // [M, runs]: token scales
  int64_t scales_row, scales_group;
  const float* weight_scales;  // [ceil(N / 128), runs]
  const void* bias;
  void* out;
  int* status;
  int64_t M;
  int N, runs;
  int ch_tiles, tok_tiles;
};

// ---------------------------------------------------------------------------------------------- PTX of this kernel
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor, kind::f8f6f4, e4m3 x e4m3 -> fp32, both operands K-major.
// Bits: [4,6) D format 1 = f32, [7,10) and [10,13) A and B format 0 = e4m3, [17,23) N >> 3, [24,29) M >> 4.
__host__ __device__ constexpr uint32_t umma_idesc_e4m3(uint32_t m, uint32_t n) {
  return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
  return static_cast<uint64_t>(lo) | (static_cast<uint64_t>(hi) << 32);
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_address(uint32_t smem_addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 load_peer(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void report_timeout(int* status, volatile int* abort_flag, int code) {
  *abort_flag = code;
  if (status != nullptr) atomicCAS(status, 0, code);
}

template <typename T>
__device__ __forceinline__ void load_bias8(const void* bias, int n, float (&b)[8]) {
  // element by element: the caller's bias may start anywhere
  const T* p = static_cast<const T*>(bias) + n;
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = static_cast<float>(__ldg(p + e));
}

// ---------------------------------------------------------------------------------------------- few tokens
__host__ __device__ constexpr int few_stages(int tok) { return tok >= 128 ? 6 : 8; }
__host__ __device__ constexpr int few_drain_warps(int tok) { return tok >= 128 ? 8 : 4; }
__host__ __device__ constexpr uint32_t few_stage_bytes(int tok) { return kRun * kRun + tok * kRun; }
__host__ __device__ constexpr uint32_t few_smem(int tok) {
  // ring + the drain warps' scale tables (two of `tok` floats each) + barriers and words, and the alignment of the ring
  return few_stages(tok) * few_stage_bytes(tok) + few_drain_warps(tok) * 2 * tok * 4 + 256 + 1024;
}

template <int TOK, typename OutT>
__global__ void __launch_bounds__(128 + 32 * few_drain_warps(TOK), 1)
    sq_fp8_few_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_weight, const Fp8Args p) {
  constexpr int S = few_stages(TOK);
  constexpr int kDrain = few_drain_warps(TOK);
  constexpr int kCols = TOK / (kDrain / 4);  // token columns of a drain warp
  constexpr int kAcc = 4;                    // accumulators in flight
  constexpr uint32_t kWBytes = kRun * kRun, kXBytes = TOK * kRun;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t w_ring = base, x_ring = base + S * kWBytes;
  const uint32_t table = x_ring + S * kXBytes;
  const uint32_t bars = table + kDrain * 2 * TOK * 4;
  const uint32_t bar_full = bars, bar_empty = bars + 8 * S, bar_acc_full = bars + 16 * S, bar_acc_empty = bar_acc_full + 8 * kAcc;
  const uint32_t words = bar_acc_empty + 8 * kAcc;
  volatile uint32_t* tmem_word = reinterpret_cast<volatile uint32_t*>(gen + (words - base));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + (words + 4 - base));

  volatile int keep_on = 0;  // an abort flag that nobody sets

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < kAcc; ++b) {
      mbar_init(bar_acc_full + 8 * b, 1);
      mbar_init(bar_acc_empty + 8 * b, kDrain);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_codes);
    tma_prefetch_desc(&map_weight);
  }
  if (warp == 2) {
    tmem_alloc(words, kAcc * TOK);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_word;

  const uint32_t parts = cluster_size(), part = cluster_rank();
  const int tile = static_cast<int>(blockIdx.x / parts);
  const int ch0 = (tile % p.ch_tiles) * kRun;
  const int64_t tok0 = static_cast<int64_t>(tile / p.ch_tiles) * TOK;
  const int g0 = static_cast<int>(static_cast<int64_t>(part) * p.runs / parts);
  const int g1 = static_cast<int>(static_cast<int64_t>(part + 1) * p.runs / parts);

  if (warp == 0) {
    // TMA producer.  The weights do not come from the kernel in front (a quantizer writes the codes and scales), so
    // the first round of weight tiles is requested before waiting for it.
    const int ahead = min(S, g1 - g0);
    if (elect_one()) {
      for (int i = 0; i < ahead; ++i) {
        mbar_arrive_expect_tx(bar_full + 8 * i, kWBytes + kXBytes);
        tma_load_2d(w_ring + i * kWBytes, &map_weight, (g0 + i) * kRun, ch0, bar_full + 8 * i);
      }
    }
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (elect_one()) {
      for (int i = 0; i < ahead; ++i)
        tma_load_2d(x_ring + i * kXBytes, &map_codes, (g0 + i) * kRun, static_cast<int32_t>(tok0), bar_full + 8 * i);
    }
    __syncwarp();
    uint32_t s = ahead == S ? 0 : ahead, phase = ahead == S ? 1 : 0, issued = ahead;
    for (int g = g0 + ahead; g < g1; ++g, ++issued) {
      if (!mbar_wait_bounded(bar_empty + 8 * s, phase ^ 1u, abort_flag, kWaitLimitNs)) {
        if (lane == 0) report_timeout(p.status, abort_flag, 9201);
        break;
      }
      if (elect_one()) {
        mbar_arrive_expect_tx(bar_full + 8 * s, kWBytes + kXBytes);
        tma_load_2d(w_ring + s * kWBytes, &map_weight, g * kRun, ch0, bar_full + 8 * s);
        tma_load_2d(x_ring + s * kXBytes, &map_codes, g * kRun, static_cast<int32_t>(tok0), bar_full + 8 * s);
      }
      __syncwarp();
      if (++s == S) {
        s = 0;
        phase ^= 1u;
      }
    }
    // no copy may be in flight when the ring is reused or the thread block leaves, after a wait that ran out either
    for (uint32_t i = issued > S ? issued - S : 0; i < issued; ++i)
      mbar_wait_bounded(bar_full + 8 * (i % S), (i / S) & 1u, &keep_on, kWaitLimitNs);
  } else if (warp == 1) {
    // MMA issuer: one accumulator per run of 128 k, four instructions of 32 k each
    uint32_t s = 0, phase = 0, acc = 0, acc_phase = 0;
    constexpr uint32_t idesc = umma_idesc_e4m3(kRun, TOK);
    uint32_t done = 0;
    for (int g = g0; g < g1; ++g, ++done) {
      if (!mbar_wait_bounded(bar_acc_empty + 8 * acc, acc_phase ^ 1u, abort_flag, kWaitLimitNs)) {
        if (lane == 0) report_timeout(p.status, abort_flag, 9202);
        break;
      }
      if (!mbar_wait_bounded(bar_full + 8 * s, phase, abort_flag, kWaitLimitNs)) {
        if (lane == 0) report_timeout(p.status, abort_flag, 9203);
        break;
      }
      tc_fence_after_sync();
      if (elect_one()) {
        const uint64_t a = umma_desc_k128(w_ring + s * kWBytes), b = umma_desc_k128(x_ring + s * kXBytes);
#pragma unroll
        for (int i = 0; i < 4; ++i) umma_f8(tmem + acc * TOK, a + 2 * i, b + 2 * i, idesc, i != 0);
        umma_commit(bar_empty + 8 * s);
        umma_commit(bar_acc_full + 8 * acc);
      }
      __syncwarp();
      if (++s == S) {
        s = 0;
        phase ^= 1u;
      }
      if (++acc == kAcc) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    // the accumulators still being written when a wait ran out: let the instructions end before the memory is freed
    for (uint32_t i = done > kAcc ? done - kAcc : 0; i < done; ++i)
      mbar_wait_bounded(bar_acc_full + 8 * (i % kAcc), (i / kAcc) & 1u, &keep_on, kWaitLimitNs);
  } else if (warp >= 4) {
    // Drain: lane = output channel, columns = tokens.  The run's scales of the warp's tokens, times the weight block's
    // scale, go through a small table (read four at a time, the same address in every lane); they are requested two
    // runs ahead.
    const int quarter = warp & 3, share = (warp - 4) >> 2;
    constexpr int kPerLane = kCols > 32 ? kCols / 32 : 1;
    float* rows = reinterpret_cast<float*>(gen + (table - base)) + (warp - 4) * 2 * TOK;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float* weight_scales = p.weight_scales + static_cast<int64_t>(ch0 / kRun) * p.runs;
    float token_scale[2][kPerLane], block_scale[2];
    auto request = [&](int g, int slot) {
      block_scale[slot] = g < g1 ? __ldg(weight_scales + g) : 0.0f;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int64_t m = tok0 + share * kCols + lane * kPerLane + i;
        token_scale[slot][i] = (lane * kPerLane < kCols && g < g1 && m < p.M) ? __ldg(p.scales + m * p.scales_row + g * p.scales_group) : 0.0f;
      }
    };
    request(g0, 0);
    request(g0 + 1, 1);
    uint64_t sums[kCols / 2];
#pragma unroll
    for (int i = 0; i < kCols / 2; ++i) sums[i] = 0;
    uint32_t acc = 0, acc_phase = 0;
    auto step = [&](int g, int slot) -> bool {
      float* mine = rows + slot * TOK;
      if (lane * kPerLane < kCols) {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) mine[lane * kPerLane + i] = token_scale[slot][i] * block_scale[slot];
      }
      request(g + 2, slot);
      __syncwarp();
      if (!mbar_wait_bounded(bar_acc_full + 8 * acc, acc_phase, abort_flag, kWaitLimitNs)) {
        if (lane == 0) report_timeout(p.status, abort_flag, 9204);
        return false;
      }
      tc_fence_after_sync();
      uint32_t d[kCols];
      tmem_ld_chunk(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * TOK + share * kCols, d);
      tmem_wait_ld_of(d);
      tc_fence_before_sync();
      if (lane == 0) mbar_arrive(bar_acc_empty + 8 * acc);
#pragma unroll
      for (int i = 0; i < kCols / 4; ++i) {
        const float4 f = *reinterpret_cast<const float4*>(mine + 4 * i);
        sums[2 * i] = ffma2(pair_of(d[4 * i], d[4 * i + 1]), pair_of(__float_as_uint(f.x), __float_as_uint(f.y)), sums[2 * i]);
        sums[2 * i + 1] = ffma2(pair_of(d[4 * i + 2], d[4 * i + 3]), pair_of(__float_as_uint(f.z), __float_as_uint(f.w)), sums[2 * i + 1]);
      }
      if (++acc == kAcc) {
        acc = 0;
        acc_phase ^= 1u;
      }
      return true;
    };
    bool ok = true;
    for (int g = g0; g < g1 && ok; g += 2) {
      ok = step(g, 0);
      if (ok && g + 1 < g1) ok = step(g + 1, 1);
    }
    // the part's sums, a token per row of 128 channels, over the ring: every copy and every MMA on it has ended (the
    // last accumulator is committed after them)
    if (ok) {
      float* sink = reinterpret_cast<float*>(gen) + quarter * 32 + lane;
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) {
        sink[(share * kCols + 2 * i) * kRun] = __uint_as_float(static_cast<uint32_t>(sums[i]));
        sink[(share * kCols + 2 * i + 1) * kRun] = __uint_as_float(static_cast<uint32_t>(sums[i] >> 32));
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  cluster_sync();
  if (warp == 2) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kAcc * TOK);
  }
  // each thread block finishes its share of the tokens: 16 chunks of 8 channels per token
  const int begin = static_cast<int>(part * TOK / parts), end = static_cast<int>((part + 1) * TOK / parts);
  for (int item = begin * 16 + static_cast<int>(threadIdx.x); item < end * 16; item += blockDim.x) {
    const int token = item >> 4, n = ch0 + (item & 15) * 8;
    if (tok0 + token >= p.M || n >= p.N) continue;
    float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const uint32_t at = base + static_cast<uint32_t>(token * kRun + (item & 15) * 8) * 4;
    for (uint32_t r = 0; r < parts; ++r) {
      const uint32_t from = peer_address(at, r);
      const float4 lo = load_peer(from), hi = load_peer(from + 16);
      y[0] += lo.x; y[1] += lo.y; y[2] += lo.z; y[3] += lo.w;
      y[4] += hi.x; y[5] += hi.y; y[6] += hi.z; y[7] += hi.w;
    }
    if (p.bias != nullptr) {
      float b[8];
      load_bias8<OutT>(p.bias, n, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] += b[e];
    }
    *reinterpret_cast<uint4*>(static_cast<OutT*>(p.out) + (tok0 + token) * p.N + n) = pack8(y, static_cast<const OutT*>(nullptr));
  }
  __syncwarp();
  if (parts > 1) cluster_sync();  // the others may still be reading this thread block's sums
}

// ---------------------------------------------------------------------------------------------- host side
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &result) == cudaSuccess &&
        result == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(sym);
  });
  return fn;
}

// [rows, row_bytes] of bytes in boxes of [box_rows, 128] with the 128-byte swizzle; what lies outside reads as zero
bool make_map(CUtensorMap* map, const void* data, uint64_t rows, uint64_t row_bytes, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {row_bytes, rows};
  const cuuint64_t strides[1] = {row_bytes};
  const cuuint32_t box[2] = {kRun, box_rows};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(data), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sm_count() {
  static int cached[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  if (cached[dev] == 0) cudaDeviceGetAttribute(&cached[dev], cudaDevAttrMultiProcessorCount, dev);
  return cached[dev] > 0 ? cached[dev] : 148;
}

// cudaFuncSetAttribute once per kernel and device
template <typename Kernel>
int allow_smem(Kernel* kernel, uint32_t bytes, bool (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && done[dev]) return SQ_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev >= 0 && dev < 64) done[dev] = true;
  return SQ_OK;
}

template <int TOK, typename OutT>
int launch_few(const Fp8GemmArgs& a, Fp8Args p, int parts, cudaStream_t stream) {
  auto kernel = sq_fp8_few_kernel<TOK, OutT>;
  static bool configured[64] = {false};
  const int ready = allow_smem(kernel, few_smem(TOK), configured);
  if (ready != SQ_OK) return ready;
  CUtensorMap map_codes, map_weight;
  if (!make_map(&map_codes, a.codes, a.M, a.K, TOK) || !make_map(&map_weight, a.weight, a.N, a.K, kRun)) return SQ_ERR_DRIVER;
  p.tok_tiles = static_cast<int>((a.M + TOK - 1) / TOK);
  const int64_t blocks = static_cast<int64_t>(p.ch_tiles) * p.tok_tiles * parts;
  if (blocks > 0x7FFFFFFF) return SQ_ERR_SHAPE;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(blocks));
  config.blockDim = dim3(128 + 32 * few_drain_warps(TOK));
  config.dynamicSmemBytes = few_smem(TOK);
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = static_cast<unsigned>(parts);
  attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = a.after_quantize ? 2 : 1;
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, map_codes, map_weight, p);
  return err == cudaSuccess ? SQ_OK : static_cast<int>(err);
}

// Thread blocks that share a tile's K: as many as keep the GPU in one wave, at most 8 (the portable cluster size).
int pick_parts(int64_t tiles, int runs, int sms) {
  int parts = 1;
  while (parts < 8 && tiles * (parts * 2) <= sms && runs >= parts * 2) parts *= 2;
  return parts;
}

template <typename OutT>
int launch_typed(const Fp8GemmArgs& a, const Fp8Args& p, cudaStream_t stream) {
  const int tok = a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= 64 ? 64 : 128;
  const int64_t tiles = static_cast<int64_t>(p.ch_tiles) * ((a.M + tok - 1) / tok);
  const int parts = pick_parts(tiles, p.runs, sm_count());
  switch (tok) {
    case 16: return launch_few<16, OutT>(a, p, parts, stream);
    case 32: return launch_few<32, OutT>(a, p, parts, stream);
    case 64: return launch_few<64, OutT>(a, p, parts, stream);
    default: return launch_few<128, OutT>(a, p, parts, stream);
  }
}

}  // namespace

int validate_fp8_gemm(const Fp8GemmArgs& a) {
  if (a.M == 0 && a.N > 0 && a.K > 0) return SQ_OK;
  if (a.codes == nullptr || a.scales == nullptr || a.weight == nullptr || a.weight_scales == nullptr || a.out == nullptr)
    return SQ_ERR_NULL;
  if (a.out_dtype != SQ_BF16 && a.out_dtype != SQ_FP16) return SQ_ERR_ENUM;
  if (a.M < 0 || a.N <= 0 || a.K <= 0 || a.N % 8 != 0 || a.K % 16 != 0) return SQ_ERR_SHAPE;
  if (a.M > (int64_t{1} << 30) || a.N > (int64_t{1} << 24) || a.K > 131072) return SQ_ERR_SHAPE;
  if (!aligned16_host(a.codes) || !aligned16_host(a.weight) || !aligned16_host(a.out)) return SQ_ERR_SHAPE;
  if (((reinterpret_cast<uintptr_t>(a.scales) | reinterpret_cast<uintptr_t>(a.weight_scales)) & 3u) != 0) return SQ_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(a.bias) & 1u) != 0) return SQ_ERR_SHAPE;
  if (a.scales_row < 0 || a.scales_group < 0) return SQ_ERR_SHAPE;
  return SQ_OK;
}

int launch_fp8_gemm(const Fp8GemmArgs& a, cudaStream_t stream) {
  const int refused = validate_fp8_gemm(a);
  if (refused != SQ_OK || a.M == 0) return refused;
  Fp8Args p = {};
  p.scales = a.scales;
  p.scales_row = a.scales_row;
  p.scales_group = a.scales_group;
  p.weight_scales = a.weight_scales;
  p.bias = a.bias;
  p.out = a.out;
  p.status = device_status_word();
  if (p.status == nullptr) return SQ_ERR_DRIVER;
  p.M = a.M;
  p.N = static_cast<int>(a.N);
  p.runs = static_cast<int>((a.K + kRun - 1) / kRun);
  p.ch_tiles = static_cast<int>((a.N + kRun - 1) / kRun);
  return a.out_dtype == SQ_BF16 ? launch_typed<__nv_bfloat16>(a, p, stream) : launch_typed<__half>(a, p, stream);
}

}  // namespace sq
