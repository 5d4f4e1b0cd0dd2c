// Linear with 4-bit weights: W[n,k] = (q[n,k] - zero[n, k / group]) * scale[n, k / group], q packed 8 to a word.
//
// Packed format.  A row is cut into blocks of 128 weights (the last one padded with zero bits); a block is 64 bytes = 16
// words, and word 4 t + i (t, i = 0..3) holds k = 32 i + 8 t ... + 7 of the block, weight 2 j in bits 4 j and weight 2 j + 1
// in bits 16 + 4 j.  So one 16-byte load gives a thread one word of each 32-weight run (groups never straddle a word), a
// mask of 0x000f000f gives a pair of neighbouring weights, and the 8 weights of a word are one 16-byte chunk of the
// unpacked row.
//
// Unpacking without conversions: for fp16, 0x6400 | q is 1024 + q and 0x6400 | q << 4 is 1024 + 16 q, so that one
// subtraction (or a multiply-add with 1 / 16) gives q - zero exactly; for bf16, 0x4300 | q is 128 + q.
//
// Two kernels.  Up to 32 tokens: w4_stream_kernel, warp-level MMAs on q - zero, exact in 16 bits, with the scale applied to
// 32-bit sums -- bound by reading the weight.  More tokens, and the gradient of the input: w4_pair_kernel, CTA-pair tcgen05
// tiles whose weight operand is unpacked into shared memory by eight warps while the tensor cores work on earlier stages.
#pragma once
#include "mp_pair_gemm.cuh"
#include "mp_stream_mma.cuh"

namespace mp {

struct W4Weight {
  const uint4* packed;       // [N][blocks][4] 16-byte chunks
  const uint16_t* scale;     // [N][groups]
  const uint8_t* zero;       // [N][groups] or null (8)
  int N, K, blocks, groups;
  int shift;                 // log2(group / 32)
};

// Two 16-bit numbers in a register: bf16 or fp16.
template <bool BF16> __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (BF16) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <bool BF16> __device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t fma2_f16(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// What unpacking needs to know of a zero point z (0..128): 128 + z (bf16) or 1024 + z and -(64 + z) (fp16), in both halves.
// Whole numbers this small sit in the mantissa: 128 + z is 0x4300 + z up to 255, 1024 + z is 0x6400 + z, and 64 + z is
// 0x5400 + 16 z while below 128 (z < 64) and 0x5800 + 8 (z - 64) from there.
struct W4Zero { uint32_t a, b; };
template <bool BF16> __device__ __forceinline__ W4Zero w4_zero(uint32_t z) {
  if constexpr (BF16) {
    // 256 (z = 128) is the next binade's first number, 0x4380, where the addition arrives by itself
    return {(0x4300u + z) * 0x10001u, 0u};
  } else {
    const uint32_t b = z < 64u ? 0xd400u + 16u * z : 0xd800u + 8u * (z - 64u);
    return {(0x6400u + z) * 0x10001u, b * 0x10001u};
  }
}
// The 8 weights of a word as q - zero: out[j] = weights 2 j and 2 j + 1.
template <bool BF16> __device__ __forceinline__ void w4_unpack(uint32_t w, const W4Zero& z, uint32_t (&out)[4]) {
  if constexpr (BF16) {
    out[0] = sub2<true>((w & 0x000f000fu) | 0x43004300u, z.a);
    out[1] = sub2<true>(((w >> 4) & 0x000f000fu) | 0x43004300u, z.a);
    out[2] = sub2<true>(((w >> 8) & 0x000f000fu) | 0x43004300u, z.a);
    out[3] = sub2<true>(((w >> 12) & 0x000f000fu) | 0x43004300u, z.a);
  } else {
    const uint32_t v = w >> 8;
    out[0] = sub2<false>((w & 0x000f000fu) | 0x64006400u, z.a);
    out[1] = fma2_f16((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, z.b);      // (1024 + 16 q) / 16 - 64 - z
    out[2] = sub2<false>((v & 0x000f000fu) | 0x64006400u, z.a);
    out[3] = fma2_f16((v & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, z.b);
  }
}

// q [N, K], one byte each -> packed words.  One thread per word; at load time only.
__global__ void w4_pack_kernel(const uint8_t* q, long long ldq, uint32_t* packed, int N, int K, int blocks) {
  const long long total = (long long)N * blocks * 16;
  for (long long x = (long long)blockIdx.x * blockDim.x + threadIdx.x; x < total; x += (long long)gridDim.x * blockDim.x) {
    const long long row = x / (blocks * 16);
    const int w = (int)(x - row * (blocks * 16)), pos = w & 15;
    const int k0 = (w >> 4) * 128 + 32 * (pos & 3) + 8 * (pos >> 2);
    uint32_t v = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k0 + e < K) v |= (uint32_t)(q[row * ldq + k0 + e] & 15) << (4 * (e >> 1) + 16 * (e & 1));
    packed[x] = v;
  }
}

// ------------------------------------------------------------------------------------------------- few tokens: streaming
// A CTA owns RT * 16 rows of W against up to 8 * NT tokens; its 8 warps take the blocks of 128 k in turn and add up in warp
// order through shared memory.  A lane loads 16 bytes of its two rows per block straight into the A fragments of the
// m16n8k16 MMA (the order of k inside a sum is free: X is loaded by the same rule).
struct W4StreamParams {
  W4Weight w;
  const uint16_t* X; long long ldx;      // T rows, 16-byte aligned
  uint16_t* Y; long long ldy;
  const uint16_t* bias;                  // may be null
  int T;
};

template <bool BF16> __device__ __forceinline__ float from16(uint16_t v) {
  if constexpr (BF16) return __bfloat162float(__ushort_as_bfloat16(v));
  else return __half2float(__ushort_as_half(v));
}
template <bool BF16> __device__ __forceinline__ uint16_t to16(float v) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  else return __half_as_ushort(__float2half_rn(v));
}

template <bool BF16, int RT, int NT, bool FINE>
__global__ void __launch_bounds__(256) w4_stream_kernel(const W4StreamParams p) {
  constexpr int U = 4 / RT;                               // blocks in flight per warp: 8 16-byte loads of W per lane
  __shared__ float red[8][RT * 16][NT * 8 + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * (RT * 16);
  const W4Weight& w = p.w;
  float acc[RT][NT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[r][n][e] = 0.0f;
  // rows past the end read the last row; their sums are not stored
  int rows[RT][2];
  const uint4* src[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      rows[r][h] = min(row0 + r * 16 + h * 8 + g, w.N - 1);
      src[r][h] = w.packed + (size_t)rows[r][h] * w.blocks * 4 + t;
    }
  uint4 cur[U][RT][2];
  const auto load = [&](uint4 (&dst)[U][RT][2], int b0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int b = b0 + 8 * u;
          dst[u][r][h] = b < w.blocks ? __ldcs(src[r][h] + (size_t)b * 4) : make_uint4(0, 0, 0, 0);
        }
  };
  load(cur, warp);
  for (int b0 = warp; b0 < w.blocks; b0 += 8 * U) {
    uint4 nxt[U][RT][2];
    load(nxt, b0 + 8 * U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = b0 + 8 * u;
      if (b >= w.blocks) break;
      const int valid = min(4, (w.K - b * 128) >> 5);     // 32-weight runs of this block that exist
      float part[RT][NT][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (FINE && i >= valid) break;
        uint4 x[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int tok = n * 8 + g;
          x[n] = (tok < p.T && i < valid) ? *reinterpret_cast<const uint4*>(p.X + (long long)tok * p.ldx + b * 128 + 32 * i + 8 * t)
                                          : make_uint4(0, 0, 0, 0);
        }
        const int gi = ((b << 2) + i) >> w.shift;         // the group of this run
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          uint32_t a[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t z = w.zero != nullptr ? (uint32_t)__ldg(w.zero + (size_t)rows[r][h] * w.groups + gi) : 8u;
            const uint4 q = cur[u][r][h];
            w4_unpack<BF16>(i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w, w4_zero<BF16>(z), a[h]);
          }
          float sc[2];
          if (FINE || i == 3) {
#pragma unroll
            for (int h = 0; h < 2; ++h) sc[h] = from16<BF16>(__ldg(w.scale + (size_t)rows[r][h] * w.groups + gi));
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (FINE || i == 0) {
#pragma unroll
              for (int e = 0; e < 4; ++e) part[r][n][e] = 0.0f;
            }
            if constexpr (BF16) {
              mma_m16n8k16_bf16(part[r][n], a[0][0], a[1][0], a[0][1], a[1][1], x[n].x, x[n].y);
              mma_m16n8k16_bf16(part[r][n], a[0][2], a[1][2], a[0][3], a[1][3], x[n].z, x[n].w);
            } else {
              mma_m16n8k16_f16(part[r][n], a[0][0], a[1][0], a[0][1], a[1][1], x[n].x, x[n].y);
              mma_m16n8k16_f16(part[r][n], a[0][2], a[1][2], a[0][3], a[1][3], x[n].z, x[n].w);
            }
            if (FINE || i == 3) {
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[r][n][e] = fmaf(sc[e >> 1], part[r][n][e], acc[r][n][e]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) cur[u][r][h] = nxt[u][r][h];
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[warp][r * 16 + (e >> 1) * 8 + g][n * 8 + 2 * t + (e & 1)] = acc[r][n][e];
  __syncthreads();
  for (int x = threadIdx.x; x < RT * 16 * NT * 8; x += 256) {
    const int row = x % (RT * 16), tok = x / (RT * 16), n = row0 + row;
    if (n >= w.N || tok >= p.T) continue;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += red[i][row][tok];
    if (p.bias != nullptr) s += from16<BF16>(p.bias[n]);
    p.Y[(long long)tok * p.ldy + n] = to16<BF16>(s);
  }
}

// ----------------------------------------------------------------------------------------- more tokens: CTA-pair tiles
// D[256 rows x bn tokens], rows = output channels (forward, contraction K) or input features (gradient, contraction N).
// A stage is 128 contraction elements: 32 KB of unpacked weight and bn / 2 token rows per CTA.  Both directions unpack the
// same thing -- 128 rows of W by one block of 128 k -- into the same swizzled lines of 64 k; forward, the lines are a K-major
// operand (line = row of D), in the gradient an MN-major one (line = contraction index).
// Warps: 0 = TMA of the tokens, 1 = MMA, 2 = TMA of the packed weight, 4..7 = epilogue, 8..15 and 16..23 = unpacking, two
// groups that take alternate stages: a stage's chain (packed bytes, conversion, stores, proxy fence, arrival) lasts about
// 1600 cycles and its MMAs 1024.
constexpr int kW4Threads = 768;
constexpr int kW4RawBytes = 128 * 64;         // packed bytes per stage and CTA
constexpr int kW4MaxRawSlots = 12;
constexpr int kW4ABytes = 128 * 256;

struct W4PairParams {
  W4Weight w;
  int grad;                     // 0: Y = X W^T, 1: dX = dY W
  int rows, T, steps;           // rows of D, tokens, contraction steps of 128
  int tiles_m, tiles_n, bn, split, steps_per_split;
  int b_wide;
  int stages, stage_bytes, raw_slots;
  int vec;                      // the scales (and zeros) of a block's runs are read in one load each
  uint16_t* out; long long ldo; // out[token][row]
  const uint16_t* bias;
  float* partial;               // split > 1: [split][T][rows_pad]
  long long ld_partial;
  int* status;
};

struct W4Unit { int tm, tn, s0, s1, slice; };
__device__ __forceinline__ W4Unit w4_unit(const W4PairParams& p, int unit) {
  W4Unit u;
  u.tn = unit % p.tiles_n;                    // neighbouring pairs share the weight's tile
  const int r = unit / p.tiles_n;
  u.slice = r % p.split;
  u.tm = r / p.split;
  u.s0 = u.slice * p.steps_per_split;
  u.s1 = min(p.steps, u.s0 + p.steps_per_split);
  return u;
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
template <int OFF> __device__ __forceinline__ uint4 ld_smem_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4+%5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr), "n"(OFF) : "memory");
  return v;
}
template <int OFF> __device__ __forceinline__ void st_smem_v4(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0+%5], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "n"(OFF) : "memory");
}
// The 8 weights of a word.
template <bool BF16> __device__ __forceinline__ uint4 w4_weights(uint32_t word, const W4Zero& zero, uint32_t scale) {
  uint32_t v[4];
  w4_unpack<BF16>(word, zero, v);
  return make_uint4(mul2<BF16>(v[0], scale), mul2<BF16>(v[1], scale), mul2<BF16>(v[2], scale), mul2<BF16>(v[3], scale));
}

// FINE: groups of 32 or 64, so the runs of a block have scales of their own.
template <bool BF16, bool FINE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kW4Threads, 1)
w4_pair_kernel(const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmW, const W4PairParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_base = smem_u32(smem);
  const int stages = p.stages;
  const uint32_t raw_base = smem_base + (uint32_t)stages * (uint32_t)p.stage_bytes;
  const int raw_slots = p.raw_slots;
  const uint32_t bar_base = raw_base + (uint32_t)raw_slots * kW4RawBytes;
  auto full_bar = [&](int s) { return bar_base + 8u * (uint32_t)s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (uint32_t)(stages + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (uint32_t)(2 * stages + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (uint32_t)(2 * stages + 2 + b); };
  auto rfull_bar = [&](int b) { return bar_base + 8u * (uint32_t)(2 * stages + 4 + b); };
  auto rempty_bar = [&](int b) { return bar_base + 8u * (uint32_t)(2 * stages + 4 + raw_slots + b); };
  const uint32_t slot_off = bar_base - smem_base + 8u * (uint32_t)(2 * stages + 4 + 2 * raw_slots);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + slot_off);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
  const int units = p.tiles_m * p.tiles_n * p.split;
  int* status = p.status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(full_bar(s), 17); mbar_init(empty_bar(s), 1); }   // 1 + 8 unpacking warps per CTA
    for (int b = 0; b < 2; ++b) { mbar_init(tfull_bar(b), 1); mbar_init(tempty_bar(b), 8); }
    for (int b = 0; b < raw_slots; ++b) { mbar_init(rfull_bar(b), 1); mbar_init(rempty_bar(b), 8); }
    mbar_fence_init();
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  cluster_sync_all();
  griddep_launch_dependents();

  const int hb = p.bn >> 1;
  if (warp == 0) {
    // ------------------------------------------------------------------------------------------------------ TMA: tokens
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int unit = pair; ok && unit < units; unit += pairs) {
        const W4Unit u = w4_unit(p, unit);
        const int b0 = u.tn * p.bn + (int)rank * hb;
        for (int st = u.s0; st < u.s1; ++st) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, status, MP_DEV_TIMEOUT_PRODUCER)) { ok = false; break; }
          if (rank == 0) mbar_arrive_expect_tx(full_bar(s), 2u * (uint32_t)(hb * 256));
          pair_load(smem_base + (uint32_t)s * (uint32_t)p.stage_bytes + kW4ABytes, &tmB, mapa_shared(full_bar(s), 0), 0, p.b_wide, hb, b0, st * 2, 2);
          if (++s == stages) { s = 0; ph ^= 1u; }
        }
      }
      for (int i = 0; ok && i < stages; ++i) {
        ok = mbar_wait(empty_bar(s), ph ^ 1u, status, MP_DEV_TIMEOUT_DRAIN);
        if (++s == stages) { s = 0; ph ^= 1u; }
      }
      if (!ok) settle_copies();
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------------------------------------------ MMA (rank 0)
    if (lane == 0 && rank == 0) {
      int s = 0;
      uint32_t ph = 0, ui = 0;
      bool ok = true;
      const uint32_t idesc = umma_idesc(1u, BF16 ? 1u : 0u, kPairRows, (uint32_t)p.bn) | ((uint32_t)p.grad << 15);
      const uint64_t a_base = p.grad ? umma_smem_desc_mn(smem_base, 16384u) : umma_smem_desc_sw128(smem_base);
      const uint64_t b_base = umma_smem_desc_sw128(smem_base) + (kW4ABytes >> 4);
      const uint32_t stage16 = (uint32_t)p.stage_bytes >> 4;
      for (int unit = pair; ok && unit < units; unit += pairs, ++ui) {
        const W4Unit u = w4_unit(p, unit);
        const uint32_t buf = ui & 1u, use = ui >> 1;
        if (!mbar_wait(tempty_bar((int)buf), (use & 1u) ^ 1u, status, MP_DEV_TIMEOUT_MMA_TMEM)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * (uint32_t)kPairMaxBN;
        for (int st = u.s0; st < u.s1; ++st) {
          if (!mbar_wait(full_bar(s), ph, status, MP_DEV_TIMEOUT_MMA_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint64_t ad = a_base + (uint64_t)((uint32_t)s * stage16), bd = b_base + (uint64_t)((uint32_t)s * stage16);
#pragma unroll
          for (uint32_t kk = 0; kk < 8; ++kk) {
            // 16 contraction elements further: 32 bytes of a K-major line (the next 16 KB block after four), 16 MN-major lines
            const uint32_t a_off = p.grad ? kk * (2048u >> 4) : (kk >> 2) * (16384u >> 4) + (kk & 3u) * 2u;
            const uint32_t b_off = (kk >> 2) * ((uint32_t)hb * 128u >> 4) + (kk & 3u) * 2u;
            umma_f16_pair(d_tmem, ad + a_off, bd + b_off, idesc, (st > u.s0 || kk > 0) ? 1u : 0u);
          }
          tc_commit_pair(empty_bar(s));
          if (++s == stages) { s = 0; ph ^= 1u; }
        }
        if (ok) tc_commit_pair(tfull_bar((int)buf));
      }
    }
  } else if (warp == 2) {
    // ----------------------------------------- TMA: packed weight, as far ahead as its own ring allows (it comes from HBM)
    if (lane == 0) {
      int rs = 0;
      uint32_t rph = 0;
      bool ok = true;
      for (int unit = pair; ok && unit < units; unit += pairs) {
        const W4Unit u = w4_unit(p, unit);
        for (int st = u.s0; st < u.s1; ++st) {
          if (!mbar_wait(rempty_bar(rs), rph ^ 1u, status, MP_DEV_TIMEOUT_PRODUCER)) { ok = false; break; }
          mbar_arrive_expect_tx(rfull_bar(rs), kW4RawBytes);
          const int blk = p.grad ? u.tm * 2 + (int)rank : st;
          const int row = p.grad ? st * 128 : u.tm * kPairRows + (int)rank * 128;
          tma_load_2d(raw_base + (uint32_t)rs * kW4RawBytes, &tmW, rfull_bar(rs), blk * 64, row);
          if (++rs == raw_slots) { rs = 0; rph ^= 1u; }
        }
      }
      if (!ok) settle_copies();
    }
  } else if (warp >= 8) {
    // -------------------------------------------------------------------------------------------------------- unpacking
    // a lane takes the 16-byte chunk t of two rows 8 apart: eight neighbouring lanes are eight rows, which the 64-byte
    // swizzle of the packed tile and the 128-byte swizzle of the operand both spread over all banks
    const int group = (warp - 8) >> 3, r0 = ((warp - 8) & 7) * 16 + (lane & 7), t = lane >> 3;
    const uint32_t raw_off = raw_base + (uint32_t)(r0 * 64 + ((t ^ ((r0 >> 1) & 3)) << 4));
    const uint32_t even_off = smem_base + (uint32_t)(r0 * 128 + ((t ^ (r0 & 7)) << 4)), odd_off = even_off ^ 64u;   // runs 0, 2 and 1, 3
    int s = group, rs = group;                          // the host gives at least two of each
    uint32_t ph = 0, rph = 0;
    const W4Weight& w = p.w;
    constexpr int R = FINE ? 4 : 1;                     // groups that a block of a row meets
    // This CTA pair's steps, one after the other across its units.
    struct Step { int unit, st; W4Unit u; };
    const auto advance = [&](Step& x) {
      if (++x.st < x.u.s1) return;
      x.unit += pairs;
      if (x.unit < units) { x.u = w4_unit(p, x.unit); x.st = x.u.s0; }
    };
    uint32_t sz[2][R];                                  // scale | zero << 16
    // Scales and zeros of the lane's two rows, a step ahead of their use.  Weights that do not exist (rows past N, runs past
    // K) get scale 0: they are zero whatever their bits say.
    const auto fetch = [&](const Step& x) {
      const int blk = p.grad ? x.u.tm * 2 + (int)rank : x.st;
      const int row = (p.grad ? x.st * 128 : x.u.tm * kPairRows + (int)rank * 128) + r0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long line = (long long)(row + 8 * h) * w.groups;
        const bool real = row + 8 * h < w.N;
        if (FINE && p.vec) {
          // groups of 32: four per block; of 64: two.  The last block of a row may have fewer, its line is still whole.
          uint32_t s0 = 0, s1 = 0, z = 0x08080808u;
          if (real && blk < w.blocks) {
            if (w.shift == 0) {
              const uint2 v = __ldg(reinterpret_cast<const uint2*>(w.scale + line + 4 * blk));
              s0 = v.x; s1 = v.y;
              if (w.zero != nullptr) z = __ldg(reinterpret_cast<const uint32_t*>(w.zero + line + 4 * blk));
            } else {
              const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(w.scale + line + 2 * blk));
              s0 = __byte_perm(v, v, 0x1010); s1 = __byte_perm(v, v, 0x3232);
              if (w.zero != nullptr) z = __byte_perm(__ldg(reinterpret_cast<const uint16_t*>(w.zero + line + 2 * blk)), 0, 0x1100);
            }
          }
          sz[h][0] = (s0 & 0xffffu) | (z & 0xffu) << 16;
          sz[h][1 % R] = (s0 >> 16) | (z & 0xff00u) << 8;
          sz[h][2 % R] = (s1 & 0xffffu) | (z & 0xff0000u);
          sz[h][3 % R] = (s1 >> 16) | (z >> 24) << 16;
        } else {
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const int run = blk * 4 + i;
            const bool there = real && run * 32 < w.K;
            const long long at = line + (run >> w.shift);
            const uint32_t z = there && w.zero != nullptr ? (uint32_t)__ldg(w.zero + at) : 8u;
            sz[h][i] = (there ? (uint32_t)__ldg(w.scale + at) : 0u) | z << 16;
          }
        }
      }
    };
    Step cur{pair, 0, {}};
    if (pair < units) {
      cur.u = w4_unit(p, pair);
      cur.st = cur.u.s0;
      if (group) advance(cur);
      if (cur.unit < units) fetch(cur);
    }
    while (cur.unit < units) {
      uint32_t scale[2][R];
      W4Zero zero[2][R];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < R; ++i) { scale[h][i] = (sz[h][i] & 0xffffu) * 0x10001u; zero[h][i] = w4_zero<BF16>(sz[h][i] >> 16); }
      Step nxt = cur;
      advance(nxt);
      if (nxt.unit < units) advance(nxt);
      if (nxt.unit < units) fetch(nxt);
      if (!mbar_wait(rfull_bar(rs), rph, status, MP_DEV_TIMEOUT_MMA_FULL)) break;
      const uint4 q0 = ld_smem_v4<0>(raw_off + (uint32_t)rs * kW4RawBytes), q1 = ld_smem_v4<512>(raw_off + (uint32_t)rs * kW4RawBytes);
      __syncwarp();
      if (lane == 0) mbar_arrive(rempty_bar(rs));
      if ((rs += 2) >= raw_slots) { rs -= raw_slots; rph ^= 1u; }
      if (!mbar_wait(empty_bar(s), ph ^ 1u, status, MP_DEV_TIMEOUT_PRODUCER)) break;
      const uint32_t ev = even_off + (uint32_t)s * (uint32_t)p.stage_bytes, od = odd_off + (uint32_t)s * (uint32_t)p.stage_bytes;
      // the weight in the operand type: one rounding of the exact product (q - zero) * scale
      st_smem_v4<0>(ev, w4_weights<BF16>(q0.x, zero[0][0], scale[0][0]));
      st_smem_v4<0>(od, w4_weights<BF16>(q0.y, zero[0][1 % R], scale[0][1 % R]));
      st_smem_v4<16384>(ev, w4_weights<BF16>(q0.z, zero[0][2 % R], scale[0][2 % R]));
      st_smem_v4<16384>(od, w4_weights<BF16>(q0.w, zero[0][3 % R], scale[0][3 % R]));
      st_smem_v4<1024>(ev, w4_weights<BF16>(q1.x, zero[1][0], scale[1][0]));
      st_smem_v4<1024>(od, w4_weights<BF16>(q1.y, zero[1][1 % R], scale[1][1 % R]));
      st_smem_v4<17408>(ev, w4_weights<BF16>(q1.z, zero[1][2 % R], scale[1][2 % R]));
      st_smem_v4<17408>(od, w4_weights<BF16>(q1.w, zero[1][3 % R], scale[1][3 % R]));
      fence_async_smem();                              // the tensor cores read through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive_pair(mapa_shared(full_bar(s), 0));
      if ((s += 2) >= stages) { s -= stages; ph ^= 1u; }
      cur = nxt;
    }
  } else if (warp >= 4) {
    // --------------------------------------------------------------------------------------------------------- epilogue
    const int quad = warp & 3;
    uint32_t ui = 0;
    for (int unit = pair; unit < units; unit += pairs, ++ui) {
      const W4Unit u = w4_unit(p, unit);
      const uint32_t buf = ui & 1u, use = ui >> 1;
      const int row = u.tm * kPairRows + (int)rank * 128 + quad * 32 + lane;
      const bool live = row < p.rows;
      const float bias = live && p.bias != nullptr ? from16<BF16>(p.bias[row]) : 0.0f;
      if (!mbar_wait(tfull_bar((int)buf), use & 1u, status, MP_DEV_TIMEOUT_EPILOGUE)) break;
      tc_fence_after();
      const uint32_t t_addr = tmem_base + buf * (uint32_t)kPairMaxBN + ((uint32_t)(quad * 32) << 16);
      const int tok0 = u.tn * p.bn, ntok = min(p.bn, p.T - tok0);
      for (int c0 = 0; c0 < ntok; c0 += 32) {
        uint32_t v[32];
        __syncwarp();
        tmem_ld_x32(t_addr + (uint32_t)c0, v);
        tmem_ld_wait();
        if (live) {
          if (p.split > 1) {
            float* o = p.partial + ((long long)u.slice * p.T + tok0 + c0) * p.ld_partial + row;
#pragma unroll
            for (int j = 0; j < 32; ++j) if (c0 + j < ntok) o[(long long)j * p.ld_partial] = __uint_as_float(v[j]);
          } else {
            uint16_t* o = p.out + (long long)(tok0 + c0) * p.ldo + row;
#pragma unroll
            for (int j = 0; j < 32; ++j) if (c0 + j < ntok) o[(long long)j * p.ldo] = to16<BF16>(__uint_as_float(v[j]) + bias);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_pair(mapa_shared(tempty_bar((int)buf), 0));
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// out[t][row] = RN16(sum over slices, in their order, + bias); four rows per thread.  Launched so that its blocks may
// start while the products finish; nothing is read before they have.
template <bool BF16>
__global__ void __launch_bounds__(256) w4_reduce_kernel(const float* partial, int split, int T, int rows, long long ld_partial,
                                                        const uint16_t* bias, uint16_t* out, long long ldo) {
  griddep_wait();
  const int quads = (int)(ld_partial >> 2);
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  if (x >= (long long)T * quads) return;
  const int t = (int)(x / quads), row = (int)(x - (long long)t * quads) * 4;
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < split; ++i) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(partial + ((long long)i * T + t) * ld_partial + row));
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
  }
  uint16_t* o = out + (long long)t * ldo + row;
  if (bias != nullptr) {
#pragma unroll
    for (int e = 0; e < 4; ++e) if (row + e < rows) v[e] += from16<BF16>(bias[row + e]);
  }
  if (row + 4 <= rows && (reinterpret_cast<uintptr_t>(o) & 7) == 0) {
    *reinterpret_cast<uint2*>(o) = make_uint2(pack16(v[0], v[1], BF16), pack16(v[2], v[3], BF16));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) if (row + e < rows) o[e] = to16<BF16>(v[e]);
  }
}

}  // namespace mp
