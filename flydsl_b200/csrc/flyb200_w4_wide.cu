// libflyb200: products of 5 and more tokens on 4-bit weights (flyb200_gemv_w4a16) on the tensor core's own operand path.
//
//   c[m, n] = epilogue(sum_g scale[n, g] * sum_{k in g} (q[n, k] - z[n, g]) * a[m, k])
//
// A block takes 128 rows of weights, on the M side of tcgen05.mma, and up to 64 tokens on its N side.  The codes come into shared
// memory by TMA, a thread per row turns them into 16-bit numbers q - z (exact) and writes them to tensor memory, which is where the
// instruction takes its first operand from; the tokens stay in shared memory as TMA brings them.  The fp32 sums of a
// group are read back from tensor memory and added to the result, times the row's scale, in registers: a thread is a row there too,
// so neither scales nor zero points travel between threads, and no weight is rounded.
//
// Bound: issue slots of the decoding.  13 instructions for 8 codes, 9 of them on the integer pipe (64 lanes a cycle and SM: 57 weights a
// cycle, the stream at the copy rate is 46), and what moves, waits and sums around them: 16 x 18944 x 8192, where every SM has one
// tile, takes 24.1 us (floor 12.2); 16 x 28672 x 8192, 1.5 tiles for an SM, 47.5.  64 x 8192 x 28672, groups of 64: 61.6 on 128 blocks, 20 SMs without
// one; on the others the integer pipe is 66 % and the issue slots 78 % busy.
// Measured against it: the warp-level instruction on codes decoded in registers takes 57.5 us for 16 x 28672 x 8192, 154 for 32 tokens.
#include "../../include/flyb200.h"
#include "gemm_kernels.cuh"
#include "host_common.h"
#include "w4.cuh"

#include <atomic>
#include <cstring>

namespace flyb200 {
namespace {

constexpr int ROWS = 128;         // of weights in a block
constexpr int STAGE_K = 256;      // inputs of a stage of the ring: 128 bytes of a row of codes
constexpr int HALF_K = 128;       // inputs that a group of decoding warps takes at a time
constexpr int HALF_COLS = HALF_K / 2;  // columns of tensor memory that they take
constexpr int SLOTS = 4;          // of them
constexpr uint32_t TMEM_COLS = 512;

struct WideParams {
  void* c;
  const void* scale;
  const uint8_t* zero;
  const void* bias;
  int M, N, K, epilogue;
  int split;  // blocks of a cluster, each with `part` stages of the inputs
  int part;
  int* status;
};

template <int NT, int G>
struct Wide {
  // Warps: sums (a thread has a row and up to 32 tokens), one of loads, two of multiplies, one of nothing, groups of four that decode.
  static constexpr int SUM_COLS = NT > 32 ? 32 : NT, SUM_WARPS = 4 * NT / SUM_COLS;
  static constexpr int LOAD_WARP = SUM_WARPS, MULTIPLY_WARP = SUM_WARPS + 1, MULTIPLIERS = 2, DECODE_WARP = SUM_WARPS + 4;
  static constexpr int DECODERS = NT > 32 ? 2 : 4;  // 2: what the registers of the sums leave
  static constexpr int THREADS = 32 * (DECODE_WARP + 4 * DECODERS);
  static constexpr int CODES = ROWS * 128, TOKENS = 4 * NT * 128;  // bytes of a stage
  static constexpr int STAGE = CODES + TOKENS;
  static constexpr int RED = NT * ROWS * 4;
  static constexpr int STAGES = (226 * 1024 - RED - 1024) / STAGE > 8 ? 8 : (226 * 1024 - RED - 1024) / STAGE;
  static constexpr int OFF_RED = STAGES * STAGE, OFF_MISC = OFF_RED + RED, BYTES = OFF_MISC + 512;
  static constexpr int GROUPS = HALF_K / G;  // of a half stage, each with NT columns of sums
  static constexpr int FIT = (static_cast<int>(TMEM_COLS) - SLOTS * HALF_COLS) / (GROUPS * NT);
  static constexpr int SETS = FIT > SLOTS ? SLOTS : FIT;  // of sums of a half stage
  static_assert(SETS >= 1 && STAGES >= 3 && BYTES <= 227 * 1024, "shared and tensor memory");
  // A wait by parity is only sound where the phase before the awaited one is known to be complete.  The two multiplying warps take the
  // even and the odd halves, each at its own pace: a group that came to half h by way of halves of the other kind (three
  // groups) could wait for half h - SLOTS before h - 2 SLOTS is multiplied, and be let through.  With two or four groups a slot is always
  // written by the same one.
  static_assert(SLOTS % DECODERS == 0 && SLOTS % MULTIPLIERS == 0, "a slot's waits follow each other in one warp");
};

// Registers -> TMEM: 32 lanes x 32 consecutive 32-bit columns.
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// First operand from tensor memory, second from shared memory.
__device__ __forceinline__ void umma_ts_f16(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Up to 32 tokens most waits find their phase complete, above that few do (64 x 8192 x 28672, groups of 64: 61.3 us by looking first, 56.9).
template <int NT>
__device__ __forceinline__ bool wait_of(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return NT > 32 ? mbar_wait_warp(bar, parity, abort_flag) : mbar_wait_soon(bar, parity, abort_flag);
}

// Roles meet at barriers in shared memory, each wait of bounded length:
//   full[stage]   codes and tokens of a stage have landed
//   empty[stage]  multiplied (a commit for each half), so decoded too
//   ready[slot]   half a stage of numbers is in tensor memory (4 warps), and the sums of the half SETS before it have left (4 warps, or 8)
//   done[slot]    multiplied (commit): the sums are there, the numbers may go
// What set the pace, one after the other (us of 16 x 18944 x 8192): three waits and commits a half in one warp of multiplies (32.9),
// two and a half (29.0), two such warps (24.1), and then
// it is the decoding: a second set of sums, a third warp of multiplies, six slots, scales by way of shared memory change nothing.
template <typename T, int G, int NT>
__global__ void __launch_bounds__(Wide<NT, G>::THREADS, 1)
    gemv_w4_wide_kernel(const __grid_constant__ CUtensorMap tm_codes, const __grid_constant__ CUtensorMap tm_tokens, const WideParams p) {
  using L = Wide<NT, G>;
  constexpr int GROUPS = L::GROUPS, THREADS = L::THREADS, SETS = L::SETS;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t full = base + L::OFF_MISC + 16, empty = full + 8 * L::STAGES, ready = empty + 8 * L::STAGES, done = ready + 8 * SLOTS;
  if ((base & 1023u) != 0) {  // the same in all blocks: nobody waits for this one
    if (threadIdx.x == 0) atomicCAS(p.status, 0, ST_SMEM_ALIGN);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 2);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(ready + 8 * s, 4 + L::SUM_WARPS);
      mbar_init(done + 8 * s, 1);
    }
    abort_flag[0] = 0;
    abort_flag[1] = 0;
    fence_mbar_init();
    prefetch_tensormap(&tm_codes);
    prefetch_tensormap(&tm_tokens);
  }
  if (warp == L::MULTIPLY_WARP) {
    tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t d0 = tmem, a0 = tmem + TMEM_COLS - SLOTS * HALF_COLS;
  pdl_wait<>();  // nothing in global memory is touched before this
  pdl_trigger();

  const int rank = static_cast<int>(blockIdx.x) % p.split, n0 = static_cast<int>(blockIdx.x) / p.split * ROWS;
  const int all = (p.K + STAGE_K - 1) / STAGE_K;
  const int s0 = min(rank * p.part, all), s1 = min(s0 + p.part, all);
  const int halves = 2 * (s1 - s0);
  const int n_groups = p.K / G;
  const int row = warp % 4 * 32 + lane;  // of sums and decoding warps
  const uint32_t quarter = static_cast<uint32_t>(warp % 4 * 32) << 16;
  float acc[L::SUM_COLS];

  if (warp == L::LOAD_WARP) {
    // ---- loads ----
    const bool issuer = elect_one();
    const uint64_t once = l2_policy_evict_first(), kept = l2_policy_evict_last();
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int s = s0; s < s1; ++s) {
      if (!wait_of<NT>(empty + 8 * stage, phase ^ 1u, abort_flag)) {
        report_failure(p.status, ST_TIMEOUT, abort_flag);
        ok = false;
        break;
      }
      if (issuer) {
        const uint32_t fb = full + 8 * stage, at = base + stage * L::STAGE;
        mbar_expect_tx(fb, L::STAGE);
        tma_load_2d(at, &tm_codes, fb, s * 128, n0, once);
#pragma unroll
        for (int b = 0; b < 4; ++b) tma_load_2d(at + L::CODES + b * NT * 128, &tm_tokens, fb, s * 512 + b * 128, 0, kept);
      }
      ++issued;
      if (++stage == L::STAGES) stage = 0, phase ^= 1u;
    }
    if (!ok || *abort_flag) {  // copies in flight land before the block leaves
      const int pending = min(issued, L::STAGES);
      for (int i = 0; i < pending; ++i) {
        int s = stage - 1 - i;
        uint32_t ph = phase;
        if (s < 0) s += L::STAGES, ph ^= 1u;
        mbar_wait(full + 8 * s, ph, abort_flag + 1);
      }
    }
  } else if (warp >= L::MULTIPLY_WARP && warp < L::MULTIPLY_WARP + L::MULTIPLIERS) {
    // ---- multiplies: of the first and of the second half of every stage ----
    const bool issuer = elect_one();
    constexpr uint32_t idesc = umma_idesc(1, W4<T>::FORMAT, ROWS, NT);
    const int mine = warp - L::MULTIPLY_WARP;
    int stage = 0, slot = mine, set = mine % SETS;
    uint32_t phase = 0, slot_phase = 0;
    for (int h = mine; h < halves; h += 2) {
      if (!wait_of<NT>(full + 8 * stage, phase, abort_flag) || !wait_of<NT>(ready + 8 * slot, slot_phase, abort_flag)) {
        report_failure(p.status, ST_TIMEOUT, abort_flag);
        break;
      }
      tc_fence_after();
      if (issuer) {
        const uint32_t tokens = base + stage * L::STAGE + L::CODES + mine * 2 * NT * 128;
#pragma unroll
        for (int k = 0; k < HALF_K / 16; ++k) {  // 16 inputs: 8 columns of numbers, 32 bytes of a token's 128
          const uint64_t bdesc = umma_desc_sw128_kmajor(tokens + (k / 4) * NT * 128) + static_cast<uint64_t>((k % 4) * 2);
          umma_ts_f16(d0 + (set * GROUPS + k * 16 / G) * NT, a0 + slot * HALF_COLS + k * 8, bdesc, idesc, k * 16 % G != 0 ? 1u : 0u);
        }
        umma_commit(done + 8 * slot);
        umma_commit(empty + 8 * stage);
      }
      if (++stage == L::STAGES) stage = 0, phase ^= 1u;
      slot += 2;
      if (slot >= SLOTS) slot -= SLOTS, slot_phase ^= 1u;
      set = (set + 2) % SETS;
    }
  } else if (warp >= L::DECODE_WARP) {
    // ---- decoding: group i takes the halves i, i + DECODERS, ...  The codes of the next one are read while the numbers of this one
    // are on their way to tensor memory. ----
    const size_t zero_row = static_cast<size_t>(min(n0 + row, p.N - 1)) * n_groups;
    int h = (warp - L::DECODE_WARP) / 4, stage = h / 2, slot = h % SLOTS;
    uint32_t phase = 0, slot_phase = 0;
    uint8_t next[GROUPS];
    auto load_zeros = [&](int half) {
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        next[j] = 8;
        if (p.zero) next[j] = __ldg(p.zero + zero_row + min((2 * s0 + half) * GROUPS + j, n_groups - 1));
      }
    };
    uint4 w[4];
    auto read_codes = [&]() {
      if (!wait_of<NT>(full + 8 * stage, phase, abort_flag)) return false;
      const uint32_t at = base + stage * L::STAGE + row * 128;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = ld_smem_v4(at + ((((h & 1) * 4 + i) ^ (row & 7)) << 4));
      return true;
    };
    bool ok = true;
    if (h < halves) {
      load_zeros(h);
      ok = read_codes();
    }
    while (h < halves && ok) {
      uint32_t offset[GROUPS];
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) offset[j] = (W4<T>::ZERO + (next[j] & 15u)) * 0x10001u;
      const int then = h + L::DECODERS;
      if (then < halves) load_zeros(then);
      if (!(ok = wait_of<NT>(done + 8 * slot, slot_phase ^ 1u, abort_flag))) break;
      tc_fence_after();
      const uint32_t dst = a0 + quarter + slot * HALF_COLS;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        uint32_t d[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint4& v = w[part * 2 + i / 4];
          const uint32_t word = i % 4 == 0 ? v.x : i % 4 == 1 ? v.y : i % 4 == 2 ? v.z : v.w;
          decode_pairs<T>(word, offset[(part * 64 + i * 8) / G], d + 4 * i);
        }
        tmem_st_x32(dst + part * 32, d);
      }
      const uint32_t written = ready + 8 * slot;
      stage += then / 2 - h / 2;
      if (stage >= L::STAGES) stage -= L::STAGES, phase ^= 1u;
      slot += L::DECODERS;
      if (slot >= SLOTS) slot -= SLOTS, slot_phase ^= 1u;
      h = then;
      if (h < halves) ok = read_codes();
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(written);
    }
    if (!ok && lane == 0) report_failure(p.status, ST_TIMEOUT, abort_flag);
  } else if (warp < L::SUM_WARPS) {
    // ---- sums ----
    const unsigned short* scale_row = static_cast<const unsigned short*>(p.scale) + static_cast<size_t>(min(n0 + row, p.N - 1)) * n_groups;
    const uint32_t sums = d0 + quarter + (warp / 4) * L::SUM_COLS;
    unsigned short next[GROUPS];
    auto load_scales = [&](int h) {
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) next[j] = __ldg(scale_row + min((2 * s0 + h) * GROUPS + j, n_groups - 1));
    };
#pragma unroll
    for (int i = 0; i < L::SUM_COLS; ++i) acc[i] = 0.0f;
    load_scales(0);
    if (lane == 0) {
      for (int h = 0; h < SETS; ++h) mbar_arrive(ready + 8 * h);
    }
    int set = 0, slot = 0, freed = SETS % SLOTS;
    uint32_t slot_phase = 0;
    for (int h = 0; h < halves; ++h) {
      float scale[GROUPS];
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) scale[j] = (2 * s0 + h) * GROUPS + j < n_groups ? W4<T>::value(next[j]) : 0.0f;
      if (h + 1 < halves) load_scales(h + 1);
      if (!wait_of<NT>(done + 8 * slot, slot_phase, abort_flag)) {
        if (lane == 0) report_failure(p.status, ST_TIMEOUT, abort_flag);
        break;
      }
      tc_fence_after();
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        const uint32_t from = sums + (set * GROUPS + j) * NT;
        uint32_t r[L::SUM_COLS];
        if constexpr (L::SUM_COLS == 16) tmem_ld_x16(from, r);
        else tmem_ld_x32(from, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < L::SUM_COLS; ++i) acc[i] = fmaf(scale[j], __uint_as_float(r[i]), acc[i]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ready + 8 * freed);
      if (++set == SETS) set = 0;
      if (++freed == SLOTS) freed = 0;
      if (++slot == SLOTS) slot = 0, slot_phase ^= 1u;
    }
  }

  // ---- the result: of a block by itself from registers, of a cluster through shared memory, added up in the order of its blocks ----
  auto store = [&](int m, int n, float v) {
    v *= W4<T>::UNIT;
    if (p.epilogue != EPI_NONE) v = w4_activation(v + W4<T>::value(static_cast<const unsigned short*>(p.bias)[n]), p.epilogue);
    static_cast<T*>(p.c)[static_cast<size_t>(m) * p.N + n] = W4<T>::round(v);
  };
  const int m0 = warp / 4 * L::SUM_COLS;  // first token of a warp of sums
  if (p.split == 1) {
    if (warp < L::SUM_WARPS && n0 + row < p.N) {
#pragma unroll
      for (int i = 0; i < L::SUM_COLS; ++i)
        if (m0 + i < p.M) store(m0 + i, n0 + row, acc[i]);
    }
  } else {
    float* red = reinterpret_cast<float*>(smem + L::OFF_RED);
    if (warp < L::SUM_WARPS) {
#pragma unroll
      for (int i = 0; i < L::SUM_COLS; ++i) red[(m0 + i) * ROWS + row] = acc[i];
    }
    __syncwarp();
    cluster_sync_all();  // also after a failed wait: every wait is bounded
    for (int i = static_cast<int>(threadIdx.x) + rank * THREADS; i < p.M * ROWS; i += p.split * THREADS) {
      if (n0 + i % ROWS >= p.N) continue;
      float v = 0.0f;
      for (int b = 0; b < p.split; ++b) v += __uint_as_float(ld_dsmem(map_to_cta(base + L::OFF_RED + 4 * i, b)));
      store(i / ROWS, n0 + i % ROWS, v);
    }
    __syncwarp();
    cluster_sync_all();  // nobody leaves while its sums are read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == L::MULTIPLY_WARP) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Blocks of a cluster: the fewest rounds of blocks times their stages; a round costs about six stages more (set-up, first bytes, sums).
// Clusters of four and eight do not cover all SMs (132 and 120 of 148).
int wide_split(int tiles, int stages) {
  const int at_once[4] = {148, 148, 132, 120};
  int best = 1;
  long long least = -1;
  for (int i = 0, split = 1; i < 4; ++i, split *= 2) {
    const int part = (stages + split - 1) / split;
    if (split > 1 && part * (split - 1) >= stages) break;  // a block without a stage
    const long long rounds = (static_cast<long long>(tiles) * split + at_once[i] - 1) / at_once[i];
    const long long cost = rounds * (part + 6) + (split > 1 ? 2 : 0);
    if (least < 0 || cost < least) least = cost, best = split;
  }
  return best;
}

template <typename T, int G, int NT>
int launch_wide(const void* a, const void* q, WideParams p, cudaStream_t s) {
  using L = Wide<NT, G>;
  auto kernel = gemv_w4_wide_kernel<T, G, NT>;
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return host::record_cuda_error(e, "cudaGetDevice");
  const uint64_t bit = 1ull << (dev & 63);
  if (!(done.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::BYTES);
    if (e != cudaSuccess) return host::record_cuda_error(e, "cudaFuncSetAttribute");
    done.fetch_or(bit, std::memory_order_release);
  }
  CUtensorMap codes, tokens;
  int rc = host::byte_matrix_map(&codes, q, p.K / 2, p.N, ROWS);
  if (!rc) rc = host::byte_matrix_map(&tokens, a, 2ull * p.K, p.M, NT);
  if (!rc) rc = host::status_word(&p.status);
  if (rc) return rc;
  const int tiles = (p.N + ROWS - 1) / ROWS, stages = (p.K + STAGE_K - 1) / STAGE_K;
  p.split = wide_split(tiles, stages);
  p.part = (stages + p.split - 1) / p.split;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles) * p.split);
  cfg.blockDim = dim3(L::THREADS);
  cfg.dynamicSmemBytes = L::BYTES;
  cfg.stream = s;
  cudaLaunchAttribute attrs[2];
  int n = 0;
  if (host::pdl_default() != 0) {
    attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.split > 1) {
    attrs[n].id = cudaLaunchAttributeClusterDimension;
    attrs[n].val.clusterDim.x = static_cast<unsigned>(p.split);
    attrs[n].val.clusterDim.y = 1;
    attrs[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attrs;
  cfg.numAttrs = n;
  e = cudaLaunchKernelEx(&cfg, kernel, codes, tokens, p);
  return e == cudaSuccess ? FLYB200_OK : host::record_cuda_error(e, "gemv_w4_wide_kernel");
}
template <typename T, int G>
int launch_wide_tokens(const void* a, const void* q, const WideParams& p, cudaStream_t s) {
  return p.M <= 16 ? launch_wide<T, G, 16>(a, q, p, s) : p.M <= 32 ? launch_wide<T, G, 32>(a, q, p, s) : launch_wide<T, G, 64>(a, q, p, s);
}

}  // namespace

namespace host {

int gemv_w4_wide(void* c, const void* a, const void* q, const void* scale, const void* zero, const void* bias, int M, int N, int K, int group,
                 bool fp16, int epilogue, void* stream) {
  WideParams p;
  memset(&p, 0, sizeof(p));
  p.c = c, p.scale = scale, p.zero = static_cast<const uint8_t*>(zero), p.bias = bias, p.M = M, p.N = N, p.K = K, p.epilogue = epilogue;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (fp16)
    return group == 32   ? launch_wide_tokens<__half, 32>(a, q, p, s)
           : group == 64 ? launch_wide_tokens<__half, 64>(a, q, p, s)
                         : launch_wide_tokens<__half, 128>(a, q, p, s);
  return group == 32   ? launch_wide_tokens<__nv_bfloat16, 32>(a, q, p, s)
         : group == 64 ? launch_wide_tokens<__nv_bfloat16, 64>(a, q, p, s)
                       : launch_wide_tokens<__nv_bfloat16, 128>(a, q, p, s);
}

}  // namespace host
}  // namespace flyb200
