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
#include "sq_overlap.h"
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
  int bias_vectors;            // the bias is 16-byte aligned
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

// Hand an accumulator back to the MMA issuer: arrive without release.  What has to come first - the warp's tensor-memory
// loads - has completed (tcgen05.wait::ld, values in registers).  A releasing arrive would also wait for the thread's
// outstanding global loads, the scales requested two runs ahead: 1000 to 1600 cycles in every run of 128 k (measured,
// 893 us instead of 469 for 8192 x 14336 x 4096).
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_peer_relaxed(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

__device__ __forceinline__ void report_timeout(int* status, volatile int* abort_flag, int code) {
  *abort_flag = code;
  if (status != nullptr) atomicCAS(status, 0, code);
}

// 8 biases, the same in every lane; one load where the caller's bias is on the vector grid
template <typename T>
__device__ __forceinline__ void load_bias8(const Fp8Args& p, int n, float (&b)[8]) {
  const T* at = static_cast<const T*>(p.bias) + n;
  if (p.bias_vectors) {
    unpack8(__ldg(reinterpret_cast<const uint4*>(at)), b, static_cast<const T*>(nullptr));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = static_cast<float>(__ldg(at + e));
  }
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
      __syncwarp();  // lanes may leave the wait one by one; the loads below are the whole warp's
      tc_fence_after_sync();
      uint32_t d[kCols];
      tmem_ld_chunk(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * TOK + share * kCols, d);
      tmem_wait_ld_of(d);
      tc_fence_before_sync();
      if (lane == 0) mbar_arrive_relaxed(bar_acc_empty + 8 * acc);
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
      load_bias8<OutT>(p, n, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] += b[e];
    }
    *reinterpret_cast<uint4*>(static_cast<OutT*>(p.out) + (tok0 + token) * p.N + n) = pack8(y, static_cast<const OutT*>(nullptr));
  }
  __syncwarp();
  if (parts > 1) cluster_sync();  // the others may still be reading this thread block's sums
}

// ---------------------------------------------------------------------------------------------- many tokens
constexpr int kPairTokens = 256;  // of a tile: 128 per thread block of the pair
constexpr int kPairThreads = 384;
constexpr int kFactorSlots = 8;
constexpr uint32_t kFactorBytes = 2 * 128 * 4;  // the factors of a run: 128 tokens for each half of the channels
constexpr int kStoreBoxes = 3;
constexpr uint32_t kStoreBytes = 32 * 32 * 2;   // a drain warp's output box: 32 tokens x 32 channels
__host__ __device__ constexpr int pair_stages(int bn) { return bn == 256 ? 5 : 7; }
__host__ __device__ constexpr uint32_t pair_stage_bytes(int bn) { return kRun * kRun + bn / 2 * kRun; }
__host__ __device__ constexpr uint32_t pair_smem(int bn) {
  return pair_stages(bn) * pair_stage_bytes(bn) + 8 * kStoreBoxes * kStoreBytes + kFactorSlots * kFactorBytes + 512 + 1024;
}

__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrive once on the barrier at this offset in both thread blocks when the MMAs issued so far are done
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(columns) : "memory");
}
// box -> this thread block's shared memory, completion on a barrier of the pair's first thread block
__device__ __forceinline__ void tma_load_pair(uint32_t dst_smem, const void* tmap, int32_t x, int32_t y, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst_smem), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(leader_bar)
      : "memory");
}

// A pair of thread blocks (cluster of two, tcgen05 cta_group::2) owns tiles of 256 tokens x BN channels: each loads its 128
// tokens and half of the channels, the tensor cores of both read both halves of the weights, and each drains its own
// 128 tokens.  A weight tile thus crosses shared memory half as often per product as with one thread block per tile,
// whose operand reads would fill the shared-memory bandwidth.
//
// Drain: lane = token, so the run's factor is ONE number per thread (token scale x weight-block scale; a warp's channels
// lie in one weight block) and an element costs one fma.  (Packed fmas made the compiler copy 90 registers per run into
// aligned pairs: 558 us against 452 for 8192 x 14336 x 4096.)  The factors are made by a warp of their own, which
// multiplies them into a ring in shared memory: loads and addresses in the drain loop cost more than the sums.
// Tensor memory holds four accumulators of 128 columns.  With BN = 256 a run is two products of 128 channels, each with
// an accumulator and four drain warps of its own, so that the tensor core has three more to work on while one is
// drained and handed back.
// Persistent: tiles are dealt out statically, loads and MMAs run ahead over tile ends, results leave through small
// swizzled boxes per warp and TMA stores.
template <int BN, typename OutT>
__global__ void __launch_bounds__(kPairThreads, 1)
    sq_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_weight,
                       const __grid_constant__ CUtensorMap map_out, const Fp8Args p) {
  constexpr int S = pair_stages(BN);
  constexpr int kParts = BN / 128;      // products of 128 channels in a run
  constexpr int kCols = BN / 2;         // channels of a drain warp
  // Batch b of four runs' factors takes the place of batch b - 2: it is written when the eight drain warps have arrived at
  // bar_factor_free for that place, each behind its last read of it.  Both barriers of a place are waited for once in each
  // of their phases by the same warps, so a phase's parity tells it from its neighbours.  (That an MMA of a later run is done
  // does not free a place: with one product a run the two issuers are not ordered, and the barrier of a run's stage may
  // still be a round behind, where the same parity has long passed.)
  static_assert(kFactorSlots == 8, "two batches of four runs");
  constexpr uint32_t kXBytes = kRun * kRun, kWBytes = BN / 2 * kRun;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t x_ring = base, w_ring = base + S * kXBytes, store_ring = w_ring + S * kWBytes;
  const uint32_t factors = store_ring + 8 * kStoreBoxes * kStoreBytes;
  const uint32_t bars = factors + kFactorSlots * kFactorBytes;
  const uint32_t bar_full = bars, bar_empty = bars + 8 * S, bar_acc_full = bars + 16 * S, bar_acc_empty = bar_acc_full + 32;
  const uint32_t bar_factor = bar_acc_empty + 32;
  const uint32_t bar_factor_free = bar_factor + 16;
  const uint32_t words = bar_factor_free + 16;
  volatile uint32_t* tmem_word = reinterpret_cast<volatile uint32_t*>(gen + (words - base));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + (words + 4 - base));
  volatile int* keep_on = reinterpret_cast<volatile int*>(gen + (words + 8 - base));  // an abort flag that nobody sets

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, kParts);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(bar_acc_full + 8 * b, 1);
      mbar_init(bar_acc_empty + 8 * b, 16 / kParts);  // the accumulator's drain warps of both thread blocks
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_factor + 8 * i, 1);
      mbar_init(bar_factor_free + 8 * i, 8);  // the drain warps of this thread block
    }
    *abort_flag = 0;
    *keep_on = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_codes);
    tma_prefetch_desc(&map_weight);
    tma_prefetch_desc(&map_out);
  }
  if (warp == 2) tmem_alloc_pair(words, 512);
  __syncwarp();
  tc_fence_before_sync();
  cluster_sync();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_word;

  const int tiles = p.ch_tiles * p.tok_tiles, pairs = static_cast<int>(gridDim.x >> 1);
  const int first = static_cast<int>(blockIdx.x >> 1);
  // tiles in strips of 8 token tiles, channels along the strip: what runs at one time shares tokens and weights in L2
  auto place = [&](int tile, int64_t& tok, int& ch) {
    const int strip = tile / (8 * p.ch_tiles), left = tile - strip * 8 * p.ch_tiles;
    const int height = min(8, p.tok_tiles - strip * 8);
    const int column = left / height;
    tok = static_cast<int64_t>(strip * 8 + left - column * height) * kPairTokens + rank * 128;
    ch = column * BN;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      // TMA producer.  Each thread block loads its own tokens and, of every product's 128 channels, 64.
      uint32_t s = 0, phase = 0, issued = 0;
      const int ahead = first < tiles ? min(S, p.runs) : 0;
      int64_t tok = 0;
      int ch = 0;
      auto load_weights = [&](uint32_t stage, int g) {
        const uint32_t bar = peer_address(bar_full + 8 * stage, 0);
        if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * stage, 2 * (kXBytes + kWBytes));
#pragma unroll
        for (int h = 0; h < kParts; ++h)
          tma_load_pair(w_ring + stage * kWBytes + h * 64 * kRun, &map_weight, g * kRun, ch + h * 128 + static_cast<int>(rank) * 64, bar);
      };
      auto load_codes = [&](uint32_t stage, int g) {
        tma_load_pair(x_ring + stage * kXBytes, &map_codes, g * kRun, static_cast<int32_t>(tok), peer_address(bar_full + 8 * stage, 0));
      };
      if (ahead > 0) {
        // the first weights do not come from the kernel in front: requested before waiting for it
        place(first, tok, ch);
        if (elect_one()) {
          for (int i = 0; i < ahead; ++i) load_weights(i, i);
        }
        __syncwarp();
      }
      asm volatile("griddepcontrol.wait;" ::: "memory");
      if (ahead > 0) {
        if (elect_one()) {
          for (int i = 0; i < ahead; ++i) load_codes(i, i);
        }
        __syncwarp();
        issued = ahead;
        s = ahead == S ? 0 : ahead;
        phase = ahead == S ? 1 : 0;
      }
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += pairs) {
        place(tile, tok, ch);
        for (int g = tile == first ? ahead : 0; g < p.runs; ++g, ++issued) {
          if (!mbar_wait_bounded(bar_empty + 8 * s, phase ^ 1u, abort_flag, kWaitLimitNs)) {
            if (lane == 0) report_timeout(p.status, abort_flag, 9211);
            ok = false;
            break;
          }
          if (elect_one()) {
            load_weights(s, g);
            load_codes(s, g);
          }
          __syncwarp();
          if (++s == S) {
            s = 0;
            phase ^= 1u;
          }
        }
      }
      // no copy may be in flight when the thread block leaves; the first one's barriers count both halves.  After a wait
      // that ran out in the second one alone there is no barrier to ask: its copies take microseconds, it waits a second.
      if (rank == 0) {
        for (uint32_t i = issued > S ? issued - S : 0; i < issued; ++i)
          mbar_wait_bounded(bar_full + 8 * (i % S), (i / S) & 1u, keep_on, kWaitLimitNs);
      } else if (!ok) {
        const uint64_t start = global_timer_ns();
        while (global_timer_ns() - start < kWaitLimitNs) asm volatile("nanosleep.u32 1000;");
      }
    } else if (warp != 2 && rank == 0) {
      // MMA issuers, for both thread blocks: two warps take the products of 128 channels in turn.  A product's two waits
      // and the issue take a warp about 500 cycles beside the drain warps on its scheduler, twice what the tensor core
      // takes for it.
      constexpr uint32_t idesc = umma_idesc_e4m3(256, 128);
      const uint32_t mine = warp >> 1;
      uint32_t s = kParts == 2 ? 0 : mine, phase = 0, acc = mine, acc_phase = 0;
      const uint64_t a0 = umma_desc_k128(x_ring), b0 = umma_desc_k128(w_ring + (kParts == 2 ? mine * 64 * kRun : 0));
      const int my_tiles = first < tiles ? (tiles - first + pairs - 1) / pairs : 0;
      const int64_t products = static_cast<int64_t>(my_tiles) * p.runs * kParts;
      int64_t at = mine;
      for (; at < products; at += 2) {
        if (!mbar_wait_bounded(bar_full + 8 * s, phase, abort_flag, kWaitLimitNs)) {
          if (lane == 0) report_timeout(p.status, abort_flag, 9213);
          break;
        }
        if (!mbar_wait_bounded(bar_acc_empty + 8 * acc, acc_phase ^ 1u, abort_flag, kWaitLimitNs)) {
          if (lane == 0) report_timeout(p.status, abort_flag, 9212);
          break;
        }
        tc_fence_after_sync();
        if (elect_one()) {
          const uint64_t a = a0 + s * (kXBytes >> 4), b = b0 + s * (kWBytes >> 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) umma_f8_pair(tmem + acc * 128, a + 2 * i, b + 2 * i, idesc, i != 0);
          umma_commit_pair(bar_acc_full + 8 * acc);
          umma_commit_pair(bar_empty + 8 * s);
        }
        __syncwarp();
        s += kParts == 2 ? 1 : 2;
        if (s >= S) {
          s -= S;
          phase ^= 1u;
        }
        acc ^= 2;
        acc_phase ^= acc == mine ? 1u : 0u;
      }
      // the accumulators still being written when a wait ran out: let the instructions end before the memory is freed
      for (int64_t i = at >= 4 ? at - 4 : mine; i < at; i += 2)
        mbar_wait_bounded(bar_acc_full + 8 * (i % 4), static_cast<uint32_t>(i / 4) & 1u, keep_on, kWaitLimitNs);
    } else if (warp == 2) {
      // Factors: four tokens and both halves' weight blocks per lane and run, in batches of four runs with one barrier each
      // (a drain warp waits for factors every fourth run).  The arrive releases the stores and waits for whatever loads
      // are under way: none, between the batches.
      asm volatile("griddepcontrol.wait;" ::: "memory");
      const int64_t rows32 = 32 * p.scales_row;
      int tile = first, g = 0, rows = 0;
      const float* token = nullptr;
      const float* block[2] = {nullptr, nullptr};
      auto aim = [&]() {
        int64_t tok;
        int ch;
        place(tile, tok, ch);
        rows = static_cast<int>(min(static_cast<int64_t>(128), p.M - tok)) - lane;  // of them 32 i < rows are there
        token = p.scales + (rows > 0 ? tok + lane : 0) * p.scales_row;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = ch + h * kCols;
          block[h] = p.weight_scales + static_cast<int64_t>(n < p.N ? n / kRun : 0) * p.runs;
        }
      };
      if (first < tiles) aim();
      uint32_t batch = 0;
      for (; tile < tiles; ++batch) {
        float t[4][4], w[4][2];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = tile < tiles;
#pragma unroll
          for (int i = 0; i < 4; ++i) t[r][i] = in && 32 * i < rows ? __ldg(token + i * rows32) : 0.0f;
#pragma unroll
          for (int h = 0; h < 2; ++h) w[r][h] = in ? __ldg(block[h] + g) : 0.0f;
          token += p.scales_group;
          if (in && ++g == p.runs) {
            g = 0;
            tile += pairs;
            if (tile < tiles) aim();
          }
        }
        if (batch >= 2 && !mbar_wait_bounded(bar_factor_free + 8 * (batch & 1u), ((batch >> 1) & 1u) ^ 1u, abort_flag, kWaitLimitNs)) {
          if (lane == 0) report_timeout(p.status, abort_flag, 9215);
          break;
        }
        const uint32_t to = factors + (batch & 1u) * 4 * kFactorBytes + lane * 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + r * kFactorBytes + h * 512 + i * 128), "f"(t[r][i] * w[r][h]) : "memory");
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_factor + 8 * (batch & 1u));
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int quarter = warp & 3, share = (warp - 4) >> 2;
    const uint32_t store = store_ring + (warp - 4) * kStoreBoxes * kStoreBytes;
    const uint32_t acc_empty = peer_address(bar_acc_empty, 0);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (kParts == 1 ? share * kCols : 0);
    const uint32_t my_factors = factors + share * 512 + (quarter * 32 + lane) * 4;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the results may overwrite what the kernel in front reads
    uint32_t acc = kParts == 1 ? 0 : share, acc_phase = 0, run = 0, box = 0;
    bool ready = false;  // the accumulator at hand was seen full while the last one was worked on
    for (int tile = first; tile < tiles; tile += pairs) {
      float sums[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) sums[i] = 0.0f;
      for (int g = 0; g < p.runs; ++g, ++run) {
        uint32_t d[2][32];
        float f;
        if (!ready && !mbar_wait_bounded(bar_acc_full + 8 * acc, acc_phase, abort_flag, kWaitLimitNs)) {
          if (lane == 0) report_timeout(p.status, abort_flag, 9214);
          goto out;
        }
        __syncwarp();
        tc_fence_after_sync();
        const uint32_t from = lanes + acc * 128;
        tmem_ld_32x32b_x32(from, d[0]);
        if ((run & 3u) == 0) {
          if (!mbar_wait_bounded(bar_factor + ((run << 1) & 8u), (run >> 3) & 1u, abort_flag, kWaitLimitNs)) {
            if (lane == 0) report_timeout(p.status, abort_flag, 9216);
            goto out;
          }
          __syncwarp();  // the wait for the loads below is the whole warp's
        }
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(my_factors + (run & 7u) * kFactorBytes) : "memory");
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          tmem_wait_ld_of(d[c & 1]);
          if (c + 1 < kCols / 32) {
            tmem_ld_32x32b_x32(from + 32 * (c + 1), d[(c + 1) & 1]);
          } else {
            tc_fence_before_sync();
            if (lane == 0) mbar_arrive_peer_relaxed(acc_empty + 8 * acc);
            acc += kParts;
            if (acc >= 4) {
              acc -= 4;
              acc_phase ^= 1u;
            }
            ready = mbar_test_wait(bar_acc_full + 8 * acc, acc_phase);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) sums[32 * c + i] = fmaf(__uint_as_float(d[c & 1][i]), f, sums[32 * c + i]);
        }
        if ((run & 3u) == 3u) {  // this warp has read the batch's factors
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_factor_free + ((run << 1) & 8u));
        }
      }
      int64_t tok;
      int ch;
      place(tile, tok, ch);
      const int64_t row0 = tok + quarter * 32;
      const int n0 = ch + share * kCols;
      // 32 channels at a time: bias, rounding, a box of 32 x 32, out by TMA (it clips what lies outside).  The box is
      // written again kStoreBoxes stores later.
#pragma unroll
      for (int part = 0; part < kCols / 32; ++part) {
        const int n = n0 + part * 32;
        uint4 packed[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = sums[part * 32 + c * 8 + e];
          if (p.bias != nullptr && n + c * 8 < p.N) {
            float b[8];
            load_bias8<OutT>(p, n + c * 8, b);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] += b[e];
          }
          packed[c] = pack8(y, static_cast<const OutT*>(nullptr));
        }
        if (lane == 0) tma_store_wait_read<kStoreBoxes - 1>();
        __syncwarp();
        const uint32_t to = store + box * kStoreBytes;
#pragma unroll
        for (int c = 0; c < 4; ++c)  // 64-byte swizzle: 16-byte chunk c of row r at c ^ (r / 2 mod 4)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                       ::"r"(to + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)), "r"(packed[c].x), "r"(packed[c].y),
                         "r"(packed[c].z), "r"(packed[c].w) : "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (n < p.N && row0 < p.M) tma_store_2d(&map_out, n, static_cast<int32_t>(row0), to);
          tma_store_commit();  // an empty group where there is nothing to store: the count of groups stays the boxes'
        }
        box = box + 1 == kStoreBoxes ? 0 : box + 1;
      }
    }
  out:
    if (lane == 0) tma_store_wait<0>();
  }
  __syncwarp();
  tc_fence_before_sync();
  cluster_sync();
  if (warp == 2) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem, 512);
  }
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

// [rows, n] of 16-bit results in boxes of [32, 32], 64-byte swizzle: what a drain warp stores
bool make_store_map(CUtensorMap* map, void* data, int dtype, uint64_t rows, uint64_t n) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {n, rows};
  const cuuint64_t strides[1] = {n * 2};
  const cuuint32_t box[2] = {32, 32};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map, dtype == SQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, data, dims, strides,
            box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
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

template <typename Kernel>
cudaLaunchConfig_t cluster_config(Kernel*, int64_t blocks, int threads, uint32_t smem, int cluster, bool after_quantize,
                                  cudaStream_t stream, cudaLaunchAttribute (&attribute)[2]) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(blocks));
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = after_quantize ? 2 : 1;
  return config;
}

template <int TOK, typename OutT>
int launch_few(const Fp8GemmArgs& a, Fp8Args p, int parts, cudaStream_t stream) {
  auto kernel = sq_fp8_few_kernel<TOK, OutT>;
  static bool configured[64] = {false};
  const int ready = allow_smem(kernel, few_smem(TOK), configured);
  if (ready != SQ_OK) return ready;
  CUtensorMap map_codes, map_weight;
  if (!make_map(&map_codes, a.codes, a.M, a.K, TOK) || !make_map(&map_weight, a.weight, a.N, a.K, kRun)) return SQ_ERR_DRIVER;
  p.ch_tiles = static_cast<int>((a.N + kRun - 1) / kRun);
  p.tok_tiles = static_cast<int>((a.M + TOK - 1) / TOK);
  const int64_t blocks = static_cast<int64_t>(p.ch_tiles) * p.tok_tiles * parts;
  if (blocks > 0x7FFFFFFF) return SQ_ERR_SHAPE;
  cudaLaunchAttribute attribute[2];
  const cudaLaunchConfig_t config = cluster_config(kernel, blocks, 128 + 32 * few_drain_warps(TOK), few_smem(TOK), parts,
                                                   a.after_quantize, stream, attribute);
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, map_codes, map_weight, p);
  return err == cudaSuccess ? SQ_OK : static_cast<int>(err);
}

template <int BN, typename OutT>
int launch_pair(const Fp8GemmArgs& a, Fp8Args p, cudaStream_t stream) {
  auto kernel = sq_fp8_pair_kernel<BN, OutT>;
  static bool configured[64] = {false};
  const int ready = allow_smem(kernel, pair_smem(BN), configured);
  if (ready != SQ_OK) return ready;
  CUtensorMap map_codes, map_weight, map_out;
  if (!make_map(&map_codes, a.codes, a.M, a.K, 128) || !make_map(&map_weight, a.weight, a.N, a.K, 64) ||
      !make_store_map(&map_out, a.out, a.out_dtype, a.M, a.N))
    return SQ_ERR_DRIVER;
  p.ch_tiles = static_cast<int>((a.N + BN - 1) / BN);
  p.tok_tiles = static_cast<int>((a.M + kPairTokens - 1) / kPairTokens);
  const int64_t tiles = static_cast<int64_t>(p.ch_tiles) * p.tok_tiles;
  if (tiles > 0x0FFFFFFF) return SQ_ERR_SHAPE;
  const int64_t pairs = tiles < sm_count() / 2 ? tiles : sm_count() / 2;
  cudaLaunchAttribute attribute[2];
  const cudaLaunchConfig_t config = cluster_config(kernel, 2 * pairs, kPairThreads, pair_smem(BN), 2, a.after_quantize, stream, attribute);
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, map_codes, map_weight, map_out, p);
  return err == cudaSuccess ? SQ_OK : static_cast<int>(err);
}

// Clusters of `parts` thread blocks with one thread block per SM that run at one time: fewer than SMs / parts where a
// GPC's SMs are no multiple of `parts` (24 clusters of 6 do not fit 148 SMs).  Asked once per device.
int cluster_capacity(int parts) {
  static int cached[64][9] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return sm_count() / parts;
  int& n = cached[dev][parts];
  if (n == 0) {
    auto kernel = sq_fp8_few_kernel<128, __nv_bfloat16>;
    static bool configured[64] = {false};
    cudaLaunchAttribute attribute[2];
    const cudaLaunchConfig_t config = cluster_config(kernel, parts, 128 + 32 * few_drain_warps(128), few_smem(128), parts, false,
                                                     nullptr, attribute);
    int found = 0;
    if (allow_smem(kernel, few_smem(128), configured) != SQ_OK || cudaOccupancyMaxActiveClusters(&found, kernel, &config) != cudaSuccess ||
        found <= 0) {
      cudaGetLastError();  // not a failure of the product: take the plain quotient
      found = sm_count() / parts;
    }
    n = found;
  }
  return n;
}

// Which kernel, tile and split: the one with the least predicted time, waves * (runs * c + e) + start, in microseconds.  The
// constants were measured on a B200 (N x K from 1024 x 14336 to 14336 x 1024, M from 1 to 2048): a run of 128 k costs a
// few-token tile of 16 / 32 / 64 / 128 tokens 0.26 / 0.27 / 0.315 / 0.42 us and a pair's tile of 256 tokens 0.235 us (128
// channels) or 0.36 us (256); a few-token tile's end costs 0.013 us per token whole and 0.022 + 0.0035 parts split.
// Predictions are within 15 % of the measured times; what they decide, with both sides measured: 128 tokens into 4096 x 1024 as
// 64-token tiles in two parts 7.1 us, as one 128-token tile 8.8; 294 tokens into 1024 x 14336 as 64-token tiles in three parts
// 19.4, as pairs 30.1; 1592 into 4096 x 4096 as pairs with 256 channels 33.8, with 128 37.1, as few-token tiles 56.7.
struct Fp8Plan {
  int tok;    // 0: a pair of thread blocks
  int parts;  // few tokens: thread blocks per tile; pair: channels
};

Fp8Plan pick_plan(int64_t M, int64_t N, int runs) {
  constexpr int kTok[4] = {16, 32, 64, 128};
  constexpr double kRunCost[4] = {0.26, 0.27, 0.315, 0.42};
  Fp8Plan best = {0, 256};
  double least = 1e30;
  for (int bn = 256; bn >= 128; bn -= 128) {
    const int64_t tiles = ((N + bn - 1) / bn) * ((M + kPairTokens - 1) / kPairTokens);
    const int64_t at_once = sm_count() / 2;
    const double cost = 4.5 + static_cast<double>((tiles + at_once - 1) / at_once) * (bn == 256 ? 0.36 * runs + 1.2 : 0.235 * runs + 0.7);
    if (cost < least) {
      least = cost;
      best = {0, bn};
    }
  }
  const int64_t channels = (N + kRun - 1) / kRun;
  for (int i = 0; i < 4; ++i) {
    const int64_t tiles = channels * ((M + kTok[i] - 1) / kTok[i]);
    for (int parts = 1; parts <= 8 && parts <= runs; ++parts) {
      const int at_once = cluster_capacity(parts);
      const double end = kTok[i] * (parts == 1 ? 0.013 : 0.022 + 0.0035 * parts);
      const double cost = 3.8 + static_cast<double>((tiles + at_once - 1) / at_once) * (kRunCost[i] * ((runs + parts - 1) / parts) + end);
      if (cost < least) {
        least = cost;
        best = {kTok[i], parts};
      }
      if (tiles > at_once) break;  // a split of tiles that fill the GPU only adds ends
    }
    if (kTok[i] >= M) break;
  }
  return best;
}

template <typename OutT>
int launch_typed(const Fp8GemmArgs& a, const Fp8Args& p, cudaStream_t stream) {
  const Fp8Plan plan = pick_plan(a.M, a.N, p.runs);
  switch (plan.tok) {
    case 16: return launch_few<16, OutT>(a, p, plan.parts, stream);
    case 32: return launch_few<32, OutT>(a, p, plan.parts, stream);
    case 64: return launch_few<64, OutT>(a, p, plan.parts, stream);
    case 128: return launch_few<128, OutT>(a, p, plan.parts, stream);
    default: break;
  }
  return plan.parts == 256 ? launch_pair<256, OutT>(a, p, stream) : launch_pair<128, OutT>(a, p, stream);
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
  const int64_t runs = (a.K + kRun - 1) / kRun;
  if (clashes(View(a.out, 2 * a.M * a.N),
              {View(a.codes, a.M * a.K), View(a.scales, 4, a.M, 4 * a.scales_row, runs, 4 * a.scales_group), View(a.weight, a.N * a.K),
               View(a.weight_scales, 4 * runs * ((a.N + kRun - 1) / kRun)), View(a.bias, 2 * a.N)}))
    return SQ_ERR_OVERLAP;
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
  p.bias_vectors = aligned16_host(a.bias);
  p.out = a.out;
  p.status = device_status_word();
  if (p.status == nullptr) return SQ_ERR_DRIVER;
  p.M = a.M;
  p.N = static_cast<int>(a.N);
  p.runs = static_cast<int>((a.K + kRun - 1) / kRun);
  return a.out_dtype == SQ_BF16 ? launch_typed<__nv_bfloat16>(a, p, stream) : launch_typed<__half>(a, p, stream);
}

}  // namespace sq
