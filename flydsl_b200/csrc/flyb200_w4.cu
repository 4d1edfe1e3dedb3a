// libflyb200: products of few tokens on 4-bit weights with a scale (and zero point) per group of inputs
// (flyb200_gemv_w4a16 in include/flyb200.h).
//
//   c[m, n] = epilogue(sum_g scale[n, g] * sum_{k in g} (q[n, k] - z[n, g]) * a[m, k])
//
// Here: the entry, and products of up to 4 tokens as integers.  More tokens: flyb200_w4_wide.cu.
// Bound: the weight stream, N K / 2 bytes; what is reached is 62 % of the copy rate (1 x 28672 x 8192 in 30.4 us, floor 18.5).  What is left
// is instructions (three for 8 codes, and the joining of limbs and scales for every group) and the last round of tiles: 896 tiles on 148 SMs are
// seven rounds for 6.05 of work, the 256 tiles of 8192 rows two for 1.73.
#include "../../include/flyb200.h"
#include "host_common.h"
#include "w4.cuh"

#include <atomic>

using namespace flyb200;

namespace {

// Tokens of a pass: up to 4 as integers below, up to 64 in flyb200_w4_wide.cu.  us, integers / wide: 1 x 28672 x 8192 30.4 / 46,
// 4 x 28672 x 8192 42.5 / 46.5, 8 x 28672 x 8192 58.5 / 46.5, 8 x 8192 x 8192 23.4 / 15.0.
constexpr int FEW_TOKENS = 4, WIDE_TOKENS = 64;
constexpr int WARPS = 16;
constexpr int CHUNK = 128;  // inputs that a warp takes at a time: 64 bytes of a row of codes

struct W4Params {
  void* c;
  const void* a;
  const uint8_t* q;
  const void* scale;
  const uint8_t* zero;
  const void* bias;
  int M, N, K, epilogue;
  int wk;        // warps that share the inputs of a row tile; WARPS / wk row tiles make a block's tile
  int tiles;     // of blocks
  int split;     // blocks of a cluster, each with `part` steps of the inputs
  int part;
  int batch;     // tiles between two meetings of the warps
  int red_at;    // bytes of shared memory ahead of the partial sums
};

// ---- asynchronous copies of 16 bytes, zeros where `in` is false ----
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
template <int WORDS>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 4) {
    const uint4 v = ld_smem_v4(a);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (WORDS == 2) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
  } else {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(a));
  }
}

// ---- up to 4 tokens: integers ------------------------------------------------------------------------------------------------
//
// The codes are multiplied as they are, as bytes: a word of 8 codes becomes two registers of four (three instructions, where
// 16-bit numbers take seven).  The activations of a group become integers of 23 bits, x = X 2^e with 2^e set by the largest
// magnitude of the group, and an integer three signed bytes ("limbs"), X = l0 + 2^8 l1 + 2^16 l2, which the instruction takes as
// three columns.  The products and their sums over a group are exact integers; what rounds is X, by 2^-22 of the group's largest
// magnitude - as much as an fp32 sum that holds it - and the fp32 sums over the groups.  An infinity or NaN makes its token NaN.
//
// Columns of an instruction: four for each token, the fourth unused; NT = 1, 2 instructions for up to 2, 4 tokens.
//
// The accumulators start at the bits of 1.5 * 2^23, so that the sum D of a column comes out as the number 1.5 * 2^23 + D.
// With its fp32 companions of a group, f = 2^e and f sum(X) of every limb, a column adds
// scale * (f D - zero f sum(X)) to the result in fp32; the limbs are put together at the end.  f is kept as a quarter, so that
// 1.5 * 2^23 f stays in range for the largest bf16 numbers, and the result is taken times 4.  For the smallest ones f is below 2^-126; it and
// its products with integers below 2^24 are exact there.
constexpr uint32_t INT_BITS = 0x4B400000u;
constexpr float INT_BASE = 12582912.0f;

constexpr int MT = 2;  // tiles of 16 rows of weights in a warp

struct IntShape {
  static constexpr int R = 16 * MT;
  static constexpr int STAGE = 1024 * MT;
  static constexpr int STAGES = 4;
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int SMEM = 227 * 1024;
  // of `steps` steps of M tokens: three bytes an activation, four floats a token and group
  static long long x_bytes(int M, int steps, int group) { return static_cast<long long>(steps) * M * (384 + CHUNK / group * 16); }
  static long long red_bytes(int M) { return static_cast<long long>(WARPS) * M * R * 4; }  // of a tile
};

__device__ __forceinline__ void imma(uint32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Position of the 8-byte chunk (8 activations of a limb) `chunk` of column `col` in its 128 bytes: without bank conflicts for the reads
// below, which take 4, 2 or 1 neighbouring chunks a lane.
template <int G>
__device__ __forceinline__ int chunk_place(int chunk, int col) {
  return chunk ^ (G == 128 ? (col & 1) << 1 : G == 64 ? (col & 1) << 3 : (col & 3) << 2);
}

// Persistent: one block per SM, in clusters of `split` blocks.  A cluster's tile is 16 MT (WARPS / wk) rows of weights; a block takes
// its part of the inputs, wk of its warps share them for 16 MT rows and take steps of 128 inputs in turn, so that neighbouring
// warps read neighbouring bytes of a row.  Each warp streams the codes of its steps, over the ends of tiles, through its own ring
// (asynchronous copies, no barrier but the warp's), and leaves the sums of a tile in shared memory; warps and blocks meet only every
// `batch` tiles, to add them up in a fixed order.
//
// Inputs in an instruction: lane (g, c) holds rows g and g + 8 of the weights and column g, and of every group the inputs
// [c G / 4, (c + 1) G / 4), that is one contiguous piece of a row of codes.  Which of the 32 input slots a code takes does not
// matter as long as the activations take the same one: a word's codes 0, 2, 4, 6 share a register, and 1, 3, 5, 7.
//
// Chunks of 16 bytes of codes are stored with their number XOR-ed by the row so that the reads of a warp meet no bank twice.
// Rows behind the last weight row are read in place of ones that do not exist; what comes out is not stored.
template <typename T, int G, int NT>
__global__ void __launch_bounds__(32 * WARPS, 1) gemv_w4_int_kernel(W4Params p) {
  using S = IntShape;
  constexpr int GROUPS = CHUNK / G;  // of a step
  constexpr int WORDS = G / 32;      // words of a lane per row and group
  constexpr int SLOTS = GROUPS * 2 * MT;  // scales that a lane needs of a step: group j, rows 16 r + 8 h + g at slot (j MT + r) 2 + h
  constexpr int LOADS = (SLOTS + 3) / 4;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait(p.c, p.a, p.q, p.scale, p.zero, p.bias);
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x % p.split, cluster = blockIdx.x / p.split, clusters = gridDim.x / p.split;
  const int n_groups = p.K / G;
  const int first = p.part * rank, last = min(first + p.part, (p.K + CHUNK - 1) / CHUNK);  // steps of this block
  const int kslot = warp & (p.wk - 1), row0 = warp / p.wk * S::R;  // of the tile
  const int tile_rows = WARPS / p.wk * S::R;
  const uint32_t ring = smem_u32(smem) + warp * S::STAGES * S::STAGE;
  const int swz = ((g >> 1) & 1) * 2 + (g >> 2);
  uint8_t* xs = smem + S::RING;                                                         // [step][3 M][128]
  float4* info = reinterpret_cast<float4*>(xs + static_cast<size_t>(last > first ? last - first : 0) * p.M * 384);  // [group][M]
  float* red = reinterpret_cast<float*>(smem + p.red_at);                               // [tile of the batch][warp][M][R]

  // codes: this lane copies chunk c of rows g + 8 i of the warp's row tile, STAGES - 1 steps ahead
  int ahead_tile = cluster, ahead = first + kslot;
  const uint8_t* q_at[2 * MT];
  auto find_codes = [&]() {
    const int n0 = ahead_tile * tile_rows + row0;
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i)
      q_at[i] = p.q + static_cast<size_t>(min(n0 + 8 * i + g, p.N - 1)) * static_cast<uint32_t>(p.K / 2) + ahead * 64 + c * 16;
  };
  uint32_t dst = ring + g * 64 + ((c ^ swz) << 4);
  const uint32_t dst_end = dst + S::STAGES * S::STAGE;
  auto copy_next = [&]() {
    if (ahead_tile < p.tiles && ahead < last) {
      if ((ahead + 1) * CHUNK <= p.K) {
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) copy16(dst + i * 512, q_at[i]);
      } else {
        const bool in = ahead * CHUNK + c * 32 < p.K;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) copy16(dst + i * 512, in ? q_at[i] : p.q, in);
      }
      dst = dst + S::STAGE == dst_end ? dst_end - S::STAGES * S::STAGE : dst + S::STAGE;
      ahead += p.wk;
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) q_at[i] += p.wk * 64;
      if (ahead >= last) {
        ahead = first + kslot;
        ahead_tile += clusters;
        find_codes();
      }
    }
    copies_commit();
  };
  // scales and zero points, one step ahead: this lane loads the slots v with v % 4 == c.  Nothing is computed on them before
  // they are used: that would wait for the loads.
  int near_tile = cluster, near = first + kslot;
  const unsigned short* s_at[LOADS];
  const uint8_t* z_at[LOADS];
  unsigned short next_scale[LOADS] = {};
  uint8_t next_zero[LOADS];
#pragma unroll
  for (int u = 0; u < LOADS; ++u) next_zero[u] = 8;
  auto find_scales = [&]() {
    const int n0 = near_tile * tile_rows + row0;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int v = 4 * u + c, r = v / 2 % MT, h = v & 1;
      const size_t e = static_cast<size_t>(min(n0 + 16 * r + 8 * h + g, p.N - 1)) * n_groups + near * GROUPS;
      s_at[u] = static_cast<const unsigned short*>(p.scale) + e;
      z_at[u] = p.zero + e;
    }
  };
  auto load_scales = [&]() {
    if (near_tile >= p.tiles || near >= last) return;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      int j = (4 * u + c) / (2 * MT) % GROUPS;
      if (GROUPS > 1) j = min(j, n_groups - 1 - near * GROUPS);  // groups behind the last one have no activations
      next_scale[u] = __ldg(s_at[u] + j);
      if (p.zero) next_zero[u] = __ldg(z_at[u] + j);
      s_at[u] += p.wk * GROUPS;
      z_at[u] += p.wk * GROUPS;
    }
    near += p.wk;
    if (near >= last) {
      near = first + kslot;
      near_tile += clusters;
      find_scales();
    }
  };
  find_codes();
  find_scales();
#pragma unroll 1
  for (int i = 0; i < S::STAGES - 1; ++i) copy_next();
  load_scales();

  // activations: a lane takes 8 of a token, the G / 8 lanes of a group are neighbours
  const int pieces = (last - first) * p.M * 16;  // a multiple of 16: the lanes of a group are in together
  auto load_piece = [&](int i) {
    const int t = i / 16 % p.M, k = (first + i / 16 / p.M) * CHUNK + (i & 15) * 8;
    return i < pieces && k < p.K ? __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.a) + static_cast<size_t>(t) * p.K + k)) : make_uint4(0u, 0u, 0u, 0u);
  };
  constexpr int DEEP = 4;  // loads in flight
  uint4 piece[DEEP];
#pragma unroll
  for (int d = 0; d < DEEP; ++d) piece[d] = load_piece(threadIdx.x + d * 32 * WARPS);
  for (int i = threadIdx.x; i < pieces; i += 32 * WARPS) {
    const int chunk = i & 15, t = i / 16 % p.M, st = i / 16 / p.M;
    const uint4 raw = piece[0];
#pragma unroll
    for (int d = 1; d < DEEP; ++d) piece[d - 1] = piece[d];
    piece[DEEP - 1] = load_piece(i + DEEP * 32 * WARPS);
    const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
    float v[8];
    uint32_t top = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = W4<T>::value(e & 1 ? in[e / 2] >> 16 : in[e / 2] & 0xFFFFu);
      top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);  // by the bits: infinities and NaN above all others
    }
    const uint32_t lanes = 0xFFFFu << (lane & 16);
#pragma unroll
    for (int o = 1; o < G / 8; o <<= 1) top = max(top, __shfl_xor_sync(lanes, top, o));
    const bool finite = top < 0x7F800000u;
    const uint32_t e = max(top >> 23, 1u);                      // max < 2^(e - 126); 2^(e - 127) <= max but for numbers below 2^-126
    const uint32_t few = e < 24u ? 24u - e : 0u;                // 2^(148 - e) in two factors where it is no fp32 number
    const float lift = __uint_as_float((127u + few) << 23);
    const float up = __uint_as_float((275u - e - few) << 23);   // |v lift up| < 2^22
    const float f = !finite ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float(e > 23u ? (e - 23u) << 23 : 1u << (e - 1u));  // 2^(e - 150)
    uint32_t u[8];
    int sum[3] = {0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t x = finite ? __float_as_uint(fmaf(v[j] * lift, up, INT_BASE)) - INT_BITS : 0u;
      u[j] = (x + 0x808080u) ^ 0x808080u;  // bytes 0, 1, 2: the limbs
    }
    uint2 limb[3];
#pragma unroll
    for (int l = 0; l < 3; ++l) {
      const uint32_t pick = l | (4 + l) << 4;
      limb[l].x = __byte_perm(__byte_perm(u[0], u[2], pick), __byte_perm(u[4], u[6], pick), 0x5410);
      limb[l].y = __byte_perm(__byte_perm(u[1], u[3], pick), __byte_perm(u[5], u[7], pick), 0x5410);
      sum[l] = __dp4a(static_cast<int>(limb[l].x), 0x01010101, __dp4a(static_cast<int>(limb[l].y), 0x01010101, 0));
      const int col = 3 * t + l;
      *reinterpret_cast<uint2*>(xs + (static_cast<size_t>(st) * 3 * p.M + col) * 128 + chunk_place<G>(chunk, col) * 8) = limb[l];
#pragma unroll
      for (int o = 1; o < G / 8; o <<= 1) sum[l] += __shfl_xor_sync(lanes, sum[l], o);
    }
    if (chunk % (G / 8) == 0)
      info[(st * GROUPS + chunk / (G / 8)) * p.M + t] = make_float4(f * static_cast<float>(sum[0]), f * static_cast<float>(sum[1]), f * static_cast<float>(sum[2]), f);
  }
  __syncthreads();

  // the lane's columns and the tokens of its sums; where there is none, another one
  uint32_t x_col[NT];
  int col[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    col[t] = 3 * min(2 * t + (g >> 2), p.M - 1) + min(g & 3, 2);
    x_col[t] = smem_u32(xs) + col[t] * 128;
  }
  uint32_t x_chunk[NT][GROUPS * (G == 128 ? 2 : 1)];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < GROUPS * (G == 128 ? 2 : 1); ++i) x_chunk[t][i] = x_col[t] + chunk_place<G>(G == 128 ? 4 * c + 2 * i : (i * 4 + c) * WORDS, col[t]) * 8;
  const float4* info_at[NT];  // of the tokens 2 t + c / 2
#pragma unroll
  for (int t = 0; t < NT; ++t) info_at[t] = info + min(2 * t + (c >> 1), p.M - 1);
  uint32_t w_chunk[GROUPS];
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    const int word = (j * 4 + c) * WORDS;  // of the row's 16
    w_chunk[j] = g * 64 + (((word >> 2) ^ swz) << 4) + (word & 3) * 4;
  }

  uint32_t stage = ring;
  int held = 0;
#pragma unroll 1
  for (int tile = cluster; tile < p.tiles; tile += clusters) {
    float acc[MT][NT][4] = {};
#pragma unroll 1
    for (int step = first + kslot; step < last; step += p.wk) {
      copies_wait<S::STAGES - 2>();
      __syncwarp();
      copy_next();  // over the stage that was read in the last round
      float scale[LOADS], zero[LOADS];
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        scale[u] = W4<T>::value(next_scale[u]);
        zero[u] = -static_cast<float>(next_zero[u] & 15);
      }
      load_scales();
      const uint32_t x_at = static_cast<uint32_t>(step - first) * p.M * 384;
      const int info_first = (step - first) * GROUPS * p.M;
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        uint32_t x[NT][WORDS][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (WORDS == 1) {
            lds_words<2>(x_chunk[t][j] + x_at, x[t][0]);
          } else {
#pragma unroll
            for (int i = 0; i < WORDS; i += 2) {
              const uint4 v = ld_smem_v4(x_chunk[t][WORDS == 4 ? i / 2 : j] + x_at);
              x[t][i][0] = v.x, x[t][i][1] = v.y, x[t][i + 1][0] = v.z, x[t][i + 1][1] = v.w;
            }
          }
        }
        float4 about[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) about[t] = info_at[t][info_first + j * p.M];
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          uint32_t sum[NT][4];
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[t][e] = INT_BITS;
          uint32_t w[2][WORDS];
#pragma unroll
          for (int h = 0; h < 2; ++h) lds_words<WORDS>(stage + (16 * r + 8 * h) * 64 + w_chunk[j], w[h]);
#pragma unroll
          for (int i = 0; i < WORDS; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              imma(sum[t], w[0][i] & 0x0F0F0F0Fu, w[1][i] & 0x0F0F0F0Fu, (w[0][i] >> 4) & 0x0F0F0F0Fu, (w[1][i] >> 4) & 0x0F0F0F0Fu, x[t][i][0], x[t][i][1]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int v = (j * MT + r) * 2 + h;
            const float s = __shfl_sync(0xffffffffu, scale[v / 4], (lane & 28) | (v & 3));
            const float z = __shfl_sync(0xffffffffu, zero[v / 4], (lane & 28) | (v & 3));
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float4& a = about[t];
                const float fx = c & 1 ? (e ? a.w : a.z) : (e ? a.y : a.x);
                acc[r][t][2 * h + e] = fmaf(s, fmaf(__uint_as_float(sum[t][2 * h + e]), a.w, fmaf(z, fx, -INT_BASE * a.w)), acc[r][t][2 * h + e]);
              }
          }
        }
      }
      stage = stage + S::STAGE == ring + S::STAGES * S::STAGE ? ring : stage + S::STAGE;
    }

    // the limbs together, and this warp's part of the tile into shared memory
    float* part = red + (held * WARPS + warp) * p.M * S::R;
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int n = 16 * r + 8 * h + g;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float v = c & 1 ? 262144.0f * acc[r][t][2 * h] : 4.0f * fmaf(256.0f, acc[r][t][2 * h + 1], acc[r][t][2 * h]);
          v += __shfl_xor_sync(0xffffffffu, v, 1);
          const int m = 2 * t + (c >> 1);
          if ((c & 1) == 0 && m < p.M) part[m * S::R + n] = v;
        }
      }
    if (++held < p.batch && tile + clusters < p.tiles) continue;

    // all sums of the batch: over the warps of a block, then over the blocks of the cluster
    const int count = held * tile_rows * p.M, first_of_batch = tile - (held - 1) * clusters;
    __syncthreads();
    if (p.split > 1) {
      for (int i = threadIdx.x; i < count; i += 32 * WARPS) {  // into the place of the first warp's
        const int n = i % tile_rows, m = i / tile_rows % p.M, b = i / tile_rows / p.M;
        float* from = red + ((b * WARPS + n / S::R * p.wk) * p.M + m) * S::R + n % S::R;
        float v = from[0];
        for (int w = 1; w < p.wk; ++w) v += from[w * p.M * S::R];
        from[0] = v;
      }
      __syncwarp();
      cluster_sync_all();
    }
    for (int i = threadIdx.x * p.split + rank; i < count; i += 32 * WARPS * p.split) {
      const int n = i % tile_rows, m = i / tile_rows % p.M, b = i / tile_rows / p.M;
      const int row = (first_of_batch + b * clusters) * tile_rows + n;
      if (row >= p.N) continue;
      const float* from = red + ((b * WARPS + n / S::R * p.wk) * p.M + m) * S::R + n % S::R;
      float v;
      if (p.split > 1) {
        const uint32_t at = smem_u32(from);
        v = 0.0f;
        for (int k = 0; k < p.split; ++k) v += __uint_as_float(ld_dsmem(map_to_cta(at, k)));
      } else {
        v = from[0];
        for (int w = 1; w < p.wk; ++w) v += from[w * p.M * S::R];
      }
      if (p.epilogue != FLYB200_EPI_NONE) v = w4_activation(v + W4<T>::value(static_cast<const unsigned short*>(p.bias)[row]), p.epilogue);
      static_cast<T*>(p.c)[static_cast<size_t>(m) * p.N + row] = W4<T>::round(v);
    }
    held = 0;
    __syncwarp();
    if (p.split > 1) cluster_sync_all();  // nobody goes on or leaves while its sums are read
    else __syncthreads();
  }
  copies_wait<0>();
}

#define CUDA_TRY(expr)                                                  \
  do {                                                                  \
    cudaError_t _e = (expr);                                            \
    if (_e != cudaSuccess) return host::record_cuda_error(_e, #expr);   \
  } while (0)

// Clusters of `split` blocks of the whole shared memory that the device runs at once: a cluster lies inside a GPC, whose SMs are not
// a multiple of every size.  Asked once per device and size.
template <typename Kernel>
cudaError_t clusters_at_once(Kernel kernel, int split, int sms, int smem, int* out) {
  static std::atomic<int> known[64][4];
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  std::atomic<int>& at = known[dev & 63][split == 1 ? 0 : split == 2 ? 1 : split == 4 ? 2 : 3];
  if (split == 1) {
    *out = sms;
    return cudaSuccess;
  }
  if ((*out = at.load()) != 0) return cudaSuccess;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(split);
  cfg.blockDim = dim3(32 * WARPS);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(split);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaError_t e = cudaOccupancyMaxActiveClusters(out, kernel, &cfg)) return e;
  if (*out < 1) *out = 1;
  at.store(*out);
  return cudaSuccess;
}

template <typename T, int G, int NT>
cudaError_t launch_int(W4Params p, int split, cudaStream_t s) {
  using S = IntShape;
  auto kernel = gemv_w4_int_kernel<T, G, NT>;
  static std::atomic<uint64_t> done{0};
  int dev = 0, sms = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  if (host::sm_count(&sms)) return cudaErrorInvalidDevice;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(done.load(std::memory_order_acquire) & bit)) {
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM)) return e;
    done.fetch_or(bit, std::memory_order_release);
  }
  const int steps = (p.K + CHUNK - 1) / CHUNK;
  p.split = split;
  p.part = (steps + split - 1) / split;
  p.wk = 1;
  while (p.wk < WARPS && 2 * p.wk <= p.part) p.wk *= 2;
  const int tile_rows = WARPS / p.wk * S::R;
  p.tiles = (p.N + tile_rows - 1) / tile_rows;
  int clusters = 0;
  if (cudaError_t e = clusters_at_once(kernel, split, sms, S::SMEM, &clusters)) return e;
  if (p.tiles < clusters) clusters = p.tiles;
  const int rounds = (p.tiles + clusters - 1) / clusters;
  const long long x = S::x_bytes(p.M, p.part, G), room = S::SMEM - S::RING - x;
  p.red_at = static_cast<int>(S::RING + x);
  const long long fit = room / S::red_bytes(p.M);
  if (fit < 1) return cudaErrorInvalidValue;
  p.batch = static_cast<int>(fit < rounds ? fit : rounds);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * split);
  cfg.blockDim = dim3(32 * WARPS);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.red_at + p.batch * S::red_bytes(p.M));
  cfg.stream = s;
  cudaLaunchAttribute attrs[2];
  int n = 0;
  if (host::pdl_default() != 0) {
    attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (split > 1) {
    attrs[n].id = cudaLaunchAttributeClusterDimension;
    attrs[n].val.clusterDim.x = static_cast<unsigned>(split);
    attrs[n].val.clusterDim.y = 1;
    attrs[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attrs;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}
// Blocks of a cluster: as few as leave room for the activations and the sums of a tile.  0: none do.
template <typename T, int G, int NT>
int split_of(const W4Params& p) {
  using S = IntShape;
  const int steps = (p.K + CHUNK - 1) / CHUNK;
  for (int split = 1; split <= 8; split *= 2) {
    const int part = (steps + split - 1) / split;
    if (part * (split - 1) >= steps && split > 1) return 0;  // a block without a step
    if (S::RING + S::x_bytes(p.M, part, G) + S::red_bytes(p.M) <= S::SMEM) return split;
  }
  return 0;
}
template <typename T, int G, int NT>
bool try_int(const W4Params& p, cudaStream_t s, cudaError_t& e) {
  const int split = split_of<T, G, NT>(p);
  if (split) e = launch_int<T, G, NT>(p, split, s);
  return split != 0;
}
// False where the activations of so many inputs do not fit.
template <typename T, int G>
bool few_tokens(const W4Params& p, cudaStream_t s, cudaError_t& e) {
  return p.M <= 2 ? try_int<T, G, 1>(p, s, e) : try_int<T, G, 2>(p, s, e);
}
template <typename T>
bool few_tokens(const W4Params& p, int group, cudaStream_t s, cudaError_t& e) {
  return group == 32 ? few_tokens<T, 32>(p, s, e) : group == 64 ? few_tokens<T, 64>(p, s, e) : few_tokens<T, 128>(p, s, e);
}

}  // namespace

extern "C" int flyb200_gemv_w4a16(void* c, const void* a, const void* q, const void* scale, const void* zero, const void* bias, int M,
                                  int N, int K, int group, int dtype, int epilogue, void* stream) {
  if (!c || !a || !q || !scale || M < 0 || N <= 0 || K <= 0) return FLYB200_E_BAD_ARG;
  if (dtype != FLYB200_DT_FP16 && dtype != FLYB200_DT_BF16) return FLYB200_E_BAD_ARG;
  if (epilogue < FLYB200_EPI_NONE || epilogue > FLYB200_EPI_BIAS_GELU || (epilogue != FLYB200_EPI_NONE && !bias)) return FLYB200_E_BAD_ARG;
  if (group != 32 && group != 64 && group != 128) return FLYB200_E_BAD_ARG;
  if (K % group != 0 || N > (1 << 27) || K > (1 << 26)) return FLYB200_E_UNSUPPORTED;
  auto multiple = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  if (!multiple(a, 16) || !multiple(q, 16) || !multiple(c, 2) || !multiple(scale, 2) || !multiple(bias, 2)) return FLYB200_E_BAD_ALIGN;
  if (M == 0) return FLYB200_OK;
  const bool fp16 = dtype == FLYB200_DT_FP16;
  for (long long m = 0; m < M; m += WIDE_TOKENS) {
    const int tokens = static_cast<int>(M - m < WIDE_TOKENS ? M - m : WIDE_TOKENS);
    char* cm = static_cast<char*>(c) + static_cast<size_t>(m) * N * 2;
    const char* am = static_cast<const char*>(a) + static_cast<size_t>(m) * K * 2;
    W4Params p = {cm, am, static_cast<const uint8_t*>(q), scale, static_cast<const uint8_t*>(zero), bias, tokens, N, K, epilogue};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (tokens <= FEW_TOKENS && (fp16 ? few_tokens<__half>(p, group, s, e) : few_tokens<__nv_bfloat16>(p, group, s, e))) {
      CUDA_TRY(e);
    } else {
      const int rc = host::gemv_w4_wide(cm, am, q, scale, zero, bias, tokens, N, K, group, fp16, epilogue, stream);
      if (rc) return rc;
    }
  }
  return FLYB200_OK;
}
