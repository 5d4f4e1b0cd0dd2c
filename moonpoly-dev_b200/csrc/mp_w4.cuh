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
// Two kernels.  Up to 16 tokens: w4_stream_kernel, warp-level MMAs on q - zero, exact in 16 bits, with the scale applied to
// 32-bit sums; its floor is reading the weight, of which it takes 2.2 times at 4 x 28672 x 4096 (21.8 us; nothing is saturated:
// latency, start and join).  More tokens, and the gradient of the input: w4_mma_kernel, tcgen05 tiles whose
// weight operand is unpacked into shared memory by sixteen warps while the tensor cores work on earlier stages.
#pragma once
#include <type_traits>

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

// What unpacking needs to know of a zero point z (0..63), in both halves: 128 + z for bf16, where 0x4300 + z is that number;
// for fp16 1024 + z, which is 0x6400 + z, and -(64 + z), which is 0xd400 + 16 z.
struct W4Zero { uint32_t a, b; };
template <bool BF16> __device__ __forceinline__ W4Zero w4_zero(uint32_t z) {
  if constexpr (BF16) return {z * 0x10001u + 0x43004300u, 0u};
  else return {z * 0x10001u + 0x64006400u, z * 0x100010u + 0xd400d400u};
}
// The exponent pattern, kept in a register: "and" with one constant and "or" with another is one instruction only if one of
// the two is a register, and the logic pipe is what the unpacking is bound by.
template <bool BF16> __device__ __forceinline__ uint32_t w4_magic() {
  uint32_t m;
  if constexpr (BF16) asm volatile("mov.b32 %0, 0x43004300;" : "=r"(m));
  else asm volatile("mov.b32 %0, 0x64006400;" : "=r"(m));
  return m;
}
template <uint32_t MASK> __device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(v), "n"(MASK), "r"(bits));
  return d;
}
// The 8 weights of a word as q - zero: out[j] = weights 2 j and 2 j + 1.
template <bool BF16> __device__ __forceinline__ void w4_unpack(uint32_t w, uint32_t magic, const W4Zero& z, uint32_t (&out)[4]) {
  if constexpr (BF16) {
    out[0] = sub2<true>(and_or<0x000f000fu>(w, magic), z.a);
    out[1] = sub2<true>(and_or<0x000f000fu>(w >> 4, magic), z.a);
    out[2] = sub2<true>(and_or<0x000f000fu>(w >> 8, magic), z.a);
    out[3] = sub2<true>(and_or<0x000f000fu>(w >> 12, magic), z.a);
  } else {
    const uint32_t v = w >> 8;
    out[0] = sub2<false>(and_or<0x000f000fu>(w, magic), z.a);
    out[1] = fma2_f16(and_or<0x00f000f0u>(w, magic), 0x2c002c00u, z.b);      // (1024 + 16 q) / 16 - 64 - z
    out[2] = sub2<false>(and_or<0x000f000fu>(v, magic), z.a);
    out[3] = fma2_f16(and_or<0x00f000f0u>(v, magic), 0x2c002c00u, z.b);
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
// One CTA of 16 warps per SM owns an equal share of the rows of W, cut into tiles of 16, against up to 8 * NT tokens.  Eight
// warps side by side take eight neighbouring blocks of 128 k of a tile -- 512 contiguous bytes of each row, which HBM
// delivers 1.3 times as fast as the 64 bytes of a warp that walks a row by itself -- and walk over the tiles first, so that
// the tokens of a block stay in registers for all of them.  The other eight warps take every other tile (or, where the share
// is a single tile, the other half of the blocks).  A (tile, warp) pair's sums wait in shared memory, 16 bytes per thread
// and eight tokens, and are added in the order of the warps at the end.
// A lane's 16 bytes of a row are the A fragments of eight m16n8k16 MMAs (the order of k inside a sum is free: X is loaded by
// the same rule), so a thread only ever uses bytes that it fetched itself: they wait in a ring of asynchronous copies in
// shared memory that no barrier guards.  Scales and zeros are brought to shared memory once, where they fit.
// The sums of a group are formed on q - zero, which is exact in 16 bits, and meet their scale in 32 bits.
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
template <int OFF> __device__ __forceinline__ uint4 ld_smem_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4+%5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr), "n"(OFF) : "memory");
  return v;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  // 0 source bytes: the 16 bytes are filled with zeros and nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
template <bool BF16> __device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&lo)[4], const uint32_t (&hi)[4], int j, uint32_t b0, uint32_t b1) {
  if constexpr (BF16) mma_m16n8k16_bf16(d, lo[j], hi[j], lo[j + 1], hi[j + 1], b0, b1);
  else mma_m16n8k16_f16(d, lo[j], hi[j], lo[j + 1], hi[j + 1], b0, b1);
}

constexpr int kW4StreamWarps = 16;

// A group's scale (low half) and zero point, as w4_zero's first half (high half), in one word.
template <bool BF16> __device__ __forceinline__ uint32_t w4_group_word(const W4Weight& w, long long at) {
  const uint32_t z = w.zero != nullptr ? (uint32_t)__ldg(w.zero + at) : 8u;
  return (uint32_t)__ldg(w.scale + at) | ((BF16 ? 0x4300u : 0x6400u) + z) << 16;
}
template <bool BF16> __device__ __forceinline__ W4Zero w4_zero_of(uint32_t word) {
  const uint32_t a = __byte_perm(word, word, 0x3232);
  return {a, BF16 ? 0u : (a & 0x003f003fu) * 16u + 0xd400d400u};
}

// GPB: groups that a block of a row meets (1, 2 or 4).  STAGED: their words are in shared memory.
template <bool BF16, int NT, int GPB, int DEPTH, bool STAGED>
__global__ void __launch_bounds__(kW4StreamWarps * 32, 1) w4_stream_kernel(const W4StreamParams p) {
  constexpr int kThreads = kW4StreamWarps * 32;
  constexpr uint32_t kSlot = kThreads * 32;               // ring bytes per block
  constexpr int G = 4 / GPB;                              // runs of 32 per group
  extern __shared__ __align__(16) uint8_t smem_raw[];
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const W4Weight& w = p.w;
  const int cta_lo = (int)((long long)w.N * blockIdx.x / gridDim.x), share = (int)((long long)w.N * (blockIdx.x + 1) / gridDim.x) - cta_lo;
  const int tiles = (share + 15) >> 4;
  const int kw = tiles > 1 ? 8 : 16, kpart = warp & (kw - 1), tile0 = warp / kw, tile_step = kW4StreamWarps / kw;
  const int outer = kpart < w.blocks && tile0 < tiles ? (w.blocks - kpart + kw - 1) / kw : 0;      // blocks of this warp
  // shared memory: ring | parked sums | group words (of whole tiles; those behind the share are whatever was there)
  uint8_t* sums = smem_raw + DEPTH * kSlot;
  uint32_t* words = reinterpret_cast<uint32_t*>(sums + (size_t)tiles * kw * (NT * 512));

  // The last tile of a share may reach into the next one's rows: they are read like any other, their sums are not stored.
  // Rows past N read as zeros.
  const uint32_t ring = smem_u32(smem_raw) + threadIdx.x * 16u;       // [slot][row half][thread]
  const long long pitch = (long long)w.blocks * 64, tile_bytes = pitch * 16 * tile_step;
  const int rows_left = w.N - cta_lo - g;                 // from this lane's first row of tile 0 on
  const uint8_t* src0 = reinterpret_cast<const uint8_t*>(w.packed) + (size_t)(cta_lo + tile0 * 16 + g) * pitch + kpart * 64 + t * 16;
  const uint8_t* src = src0;
  int b_in = outer > 0 ? kpart : w.blocks, tile_in = tile0;
  const auto issue = [&](uint32_t slot) {
    if (b_in < w.blocks) {
      const bool lo = tile_in * 16 < rows_left, hi = tile_in * 16 + 8 < rows_left;
      cp_async16(ring + slot * kSlot, lo ? src : reinterpret_cast<const uint8_t*>(w.packed), lo);
      cp_async16(ring + slot * kSlot + kThreads * 16u, hi ? src + 8 * pitch : reinterpret_cast<const uint8_t*>(w.packed), hi);
      src += tile_bytes;
      tile_in += tile_step;
      if (tile_in >= tiles) { tile_in = tile0; b_in += kw; src0 += kw * 64; src = src0; }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  griddep_wait();
#pragma unroll
  for (uint32_t d = 0; d < DEPTH; ++d) issue(d);
  const long long group_base = (long long)cta_lo * w.groups;
  if constexpr (STAGED) {
    const int num = share * w.groups;
    const uint16_t* sc = w.scale + group_base;
    const uint8_t* zr = w.zero + group_base;
    if (((reinterpret_cast<uintptr_t>(sc) & 15) | (w.zero != nullptr ? reinterpret_cast<uintptr_t>(zr) & 7 : 0) | (num & 7)) == 0) {
      for (int i = threadIdx.x * 8; i < num; i += kThreads * 8) {     // 8 groups per thread
        const uint4 s8 = __ldg(reinterpret_cast<const uint4*>(sc + i));
        const uint2 z8 = w.zero != nullptr ? __ldg(reinterpret_cast<const uint2*>(zr + i)) : make_uint2(0x08080808u, 0x08080808u);
        const uint32_t sv[4] = {s8.x, s8.y, s8.z, s8.w}, zv[2] = {z8.x, z8.y};
        uint32_t o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          o[e] = __byte_perm(sv[e >> 1], (BF16 ? 0x4300u : 0x6400u) + ((zv[e >> 2] >> (8 * (e & 3))) & 0xffu), e & 1 ? 0x5432 : 0x5410);
        reinterpret_cast<uint4*>(words + i)[0] = make_uint4(o[0], o[1], o[2], o[3]);
        reinterpret_cast<uint4*>(words + i)[1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
    } else {
      for (int i = threadIdx.x; i < num; i += kThreads) words[i] = w4_group_word<BF16>(w, group_base + i);
    }
  }

  const uint16_t* xp[NT];                                 // columns past T repeat the last token; they are not stored
#pragma unroll
  for (int n = 0; n < NT; ++n) xp[n] = p.X + (long long)min(n * 8 + g, p.T - 1) * p.ldx + 8 * t;
  uint4 x[4][NT];
  const auto load_x = [&](uint4 (&v)[4][NT], int b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = min(b * 128 + 32 * i, w.K - 32);      // a run past K is not used
#pragma unroll
      for (int n = 0; n < NT; ++n) v[i][n] = *reinterpret_cast<const uint4*>(xp[n] + k);
    }
  };
  if (outer > 0) load_x(x, kpart);
  if constexpr (STAGED) __syncthreads();

  const uint32_t magic = w4_magic<BF16>();
  uint32_t slot = 0;
  for (int o = 0; o < outer; ++o) {
    const int b = kpart + o * kw;
    const int valid = (w.K - b * 128) >> 5;               // runs of this block that exist, if fewer than 4
    const int group0 = GPB == 1 ? (b * 4) >> w.shift : b * GPB;
    uint4 xn[4][NT];
    if constexpr (NT == 1) load_x(xn, min(b + kw, w.blocks - 1));
    else if (o > 0) load_x(x, b);
    // this warp's tiles, 16 rows each, against this block; WHOLE: all four runs exist
    const auto tile_block = [&](auto whole, auto start) {
      constexpr bool WHOLE = decltype(whole)::value, START = decltype(start)::value;
      uint4* park = reinterpret_cast<uint4*>(sums) + (size_t)(tile0 * kw + kpart) * (NT * 32) + lane;
      int at_lo = (tile0 * 16 + g) * w.groups + group0;
      for (int tile = tile0; tile < tiles; tile += tile_step, park += tile_step * kw * (NT * 32), at_lo += tile_step * 16 * w.groups) {
      const int at_hi = at_lo + 8 * w.groups;
      float acc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 v = START ? make_uint4(0, 0, 0, 0) : park[n * 32];
        acc[n][0] = __uint_as_float(v.x); acc[n][1] = __uint_as_float(v.y); acc[n][2] = __uint_as_float(v.z); acc[n][3] = __uint_as_float(v.w);
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
      const uint4 q_lo = ld_smem_v4<0>(ring + slot * kSlot), q_hi = ld_smem_v4<kThreads * 16>(ring + slot * kSlot);
#pragma unroll
      for (int gi = 0; gi < GPB; ++gi) {
        if (!WHOLE && gi * G >= valid) break;
        uint32_t word_lo, word_hi;
        if constexpr (STAGED) { word_lo = words[at_lo + gi]; word_hi = words[at_hi + gi]; }
        else {                                             // rows past N: any word will do
          word_lo = tile * 16 < rows_left ? w4_group_word<BF16>(w, group_base + at_lo + gi) : 0u;
          word_hi = tile * 16 + 8 < rows_left ? w4_group_word<BF16>(w, group_base + at_hi + gi) : 0u;
        }
        const W4Zero z_lo = w4_zero_of<BF16>(word_lo), z_hi = w4_zero_of<BF16>(word_hi);
        float part[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) part[n][0] = part[n][1] = part[n][2] = part[n][3] = 0.0f;
#pragma unroll
        for (int i = gi * G; i < gi * G + G; ++i) {
          if (!WHOLE && i >= valid) break;
          uint32_t a_lo[4], a_hi[4];
          w4_unpack<BF16>(i == 0 ? q_lo.x : i == 1 ? q_lo.y : i == 2 ? q_lo.z : q_lo.w, magic, z_lo, a_lo);
          w4_unpack<BF16>(i == 0 ? q_hi.x : i == 1 ? q_hi.y : i == 2 ? q_hi.z : q_hi.w, magic, z_hi, a_hi);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma16<BF16>(part[n], a_lo, a_hi, 0, x[i][n].x, x[i][n].y);
            mma16<BF16>(part[n], a_lo, a_hi, 2, x[i][n].z, x[i][n].w);
          }
        }
        const float s_lo = from16<BF16>((uint16_t)word_lo), s_hi = from16<BF16>((uint16_t)word_hi);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[n][0] = fmaf(s_lo, part[n][0], acc[n][0]);
          acc[n][1] = fmaf(s_lo, part[n][1], acc[n][1]);
          acc[n][2] = fmaf(s_hi, part[n][2], acc[n][2]);
          acc[n][3] = fmaf(s_hi, part[n][3], acc[n][3]);
        }
      }
      issue(slot);                                         // the slot's bytes have been read by their only reader
      slot = (slot + 1) & (DEPTH - 1);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        park[n * 32] = make_uint4(__float_as_uint(acc[n][0]), __float_as_uint(acc[n][1]), __float_as_uint(acc[n][2]), __float_as_uint(acc[n][3]));
      }
    };
    if (valid < 4) {
      if (o == 0) tile_block(std::false_type{}, std::true_type{});
      else tile_block(std::false_type{}, std::false_type{});
    } else if (o == 0) {
      tile_block(std::true_type{}, std::true_type{});
    } else {
      tile_block(std::true_type{}, std::false_type{});
    }
    if constexpr (NT == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i][0] = xn[i][0];
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  const int rows = tiles * 16, parts = min(kw, w.blocks);  // warps beyond the blocks parked nothing
  const float* parked = reinterpret_cast<const float*>(sums);
  const int toks = min(p.T, NT * 8);
  for (int i = threadIdx.x; i < rows * toks; i += kThreads) {
    const int row = i % rows, tok = i / rows, n = cta_lo + row, rr = row & 15;
    if (row >= share) continue;
    const float* q = parked + (size_t)(row >> 4) * kw * (NT * 128) + (tok >> 3) * 128 + ((rr & 7) * 4 + ((tok & 7) >> 1)) * 4 + (rr >> 3) * 2 + (tok & 1);
    float s = 0.0f;
    for (int k = 0; k < parts; ++k) s += q[k * (NT * 128)];
    if (p.bias != nullptr) s += from16<BF16>(p.bias[n]);
    p.Y[(long long)tok * p.ldy + n] = to16<BF16>(s);
  }
}

// ------------------------------------------------------------------------------------------------ more tokens: tcgen05
// D[rows x bn tokens], rows = output channels (forward, contraction K) or input features (gradient, contraction N): tiles of
// 256 x bn on CTA pairs (cta_group::2), 128 rows of the weight and half of the tokens per CTA.
// A step is 128 contraction elements: 32 KB of unpacked weight and bn / 2 token rows of 256 bytes per CTA.  Both directions
// unpack the same thing -- 128 rows of W by one block of 128 k -- into the same swizzled lines of 64 k; forward, the lines are
// a K-major operand (line = row of D), in the gradient an MN-major one (line = contraction index).
// Warps: 0 = TMA of the tokens, 1 = MMA, 2 = TMA of the packed weight, 4..7 = epilogue, 8..15 and 16..23 = unpacking, two
// groups that take turns of two steps.
// Bound: up to 128 tokens by the unpacking (900 cycles of a step's two turns at 2100 warp instructions), from 256 on by the
// tensor cores (1024 cycles a step).  Tiles of single CTAs (128 x bn) were 3 to 8 % faster at 33 and 64 tokens and 9 % slower
// at 128 x 28672 x 4096, and went.
constexpr int kW4Threads = 768;
constexpr int kW4RawBytes = 2 * 128 * 64;     // packed bytes per turn and CTA
constexpr int kW4MaxRawSlots = 6;
constexpr int kW4ABytes = 128 * 256;

struct W4PairParams {
  W4Weight w;
  int grad;                     // 0: Y = X W^T, 1: dX = dY W
  int rows, T, steps;           // rows of D, tokens, contraction steps of 128
  int tiles_m, tiles_n, bn, split, steps_per_split;
  int b_wide;                   // whole blocks of 64 along the tokens' lines
  int stages, stage_bytes, raw_slots;
  const uint32_t* table; int ld_table;   // group words [groups][rows of W] (w4_table_kernel); null: scales and zeros as given
  uint16_t* out; long long ldo; // out[token][row]
  const uint16_t* bias;
  float* partial;               // split > 1: [split][T][rows_pad]
  long long ld_partial;
  int* status;
};

struct W4Unit { int tm, tn, s0, s1, slice; };
__device__ __forceinline__ W4Unit w4_unit(const W4PairParams& p, int unit) {
  W4Unit u;
  u.tn = unit % p.tiles_n;                    // neighbours share the weight's tile
  const int r = unit / p.tiles_n;
  u.slice = r % p.split;
  u.tm = r / p.split;
  u.s0 = u.slice * p.steps_per_split;
  u.s1 = min(p.steps, u.s0 + p.steps_per_split);
  return u;
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
template <int OFF> __device__ __forceinline__ void st_smem_v4(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0+%5], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "n"(OFF) : "memory");
}
// The 8 weights of a word.
template <bool BF16> __device__ __forceinline__ uint4 w4_weights(uint32_t word, uint32_t magic, const W4Zero& zero, uint32_t scale) {
  uint32_t v[4];
  w4_unpack<BF16>(word, magic, zero, v);
  return make_uint4(mul2<BF16>(v[0], scale), mul2<BF16>(v[1], scale), mul2<BF16>(v[2], scale), mul2<BF16>(v[3], scale));
}

// Scale and zero of every group as one word, scale | zero << 16, transposed to [groups][rows]: the unpacking warps read a
// step's 128 rows, and rows are neighbours only this way round.  Where they lie, [rows][groups], a step touches 256 lines of
// L1 for 512 bytes: the gradient of 4096 x 28672 x 4096 with groups of 64 took 929 us instead of 715.
__global__ void __launch_bounds__(256) w4_table_kernel(const uint16_t* scale, const uint8_t* zero, int N, int groups, int across, uint32_t* table,
                                                       int ld_table) {
  __shared__ uint32_t tile[32][33];
  griddep_launch_dependents();
  griddep_wait();
  const int n0 = (int)blockIdx.x % across * 32, g0 = (int)blockIdx.x / across * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = ty; i < 32; i += 8)
    if (n0 + i < N && g0 + tx < groups) {
      const long long at = (long long)(n0 + i) * groups + g0 + tx;
      tile[i][tx] = (uint32_t)scale[at] | (zero != nullptr ? (uint32_t)zero[at] : 8u) << 16;
    }
  __syncthreads();
  for (int i = ty; i < 32; i += 8)
    if (g0 + i < groups && n0 + tx < N) table[(long long)(g0 + i) * ld_table + n0 + tx] = tile[tx][i];
}

// FINE: groups of 32 or 64, so the runs of a block have scales of their own.
template <bool BF16, bool FINE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kW4Threads, 1)
w4_mma_kernel(const __grid_constant__ OperandMaps tokens, const __grid_constant__ CUtensorMap tmW, const W4PairParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_base = smem_u32(smem);
  const int stages = p.stages, raw_slots = p.raw_slots;
  const uint32_t raw_base = smem_base + (uint32_t)stages * (uint32_t)p.stage_bytes;
  const uint32_t bar_base = raw_base + (uint32_t)raw_slots * kW4RawBytes;
  auto full_bar = [&](int s) { return bar_base + 8u * (uint32_t)s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (uint32_t)(stages + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (uint32_t)(2 * stages + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (uint32_t)(2 * stages + 2 + b); };
  auto rfull_bar = [&](int b) { return bar_base + 8u * (uint32_t)(2 * stages + 4 + b); };
  auto rempty_bar = [&](int b) { return bar_base + 8u * (uint32_t)(2 * stages + 4 + raw_slots + b); };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + (bar_base - smem_base) + 8u * (uint32_t)(2 * stages + 4 + 2 * raw_slots));
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int first = (int)blockIdx.x >> 1, stride = (int)gridDim.x >> 1;       // units of this pair
  const int units = p.tiles_m * p.tiles_n * p.split;
  int* status = p.status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(full_bar(s), 17); mbar_init(empty_bar(s), 1); }   // 1 + 8 unpacking warps per CTA
    for (int b = 0; b < 2; ++b) { mbar_init(tfull_bar(b), 1); mbar_init(tempty_bar(b), 8); }
    for (int b = 0; b < raw_slots; ++b) { mbar_init(rfull_bar(b), 1); mbar_init(rempty_bar(b), 8); }
    mbar_fence_init();
    tma_prefetch_desc(&tokens.wide);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  cluster_sync_all();
  // Everything above may overlap the previous kernel of the stream; nothing of it is read or overwritten before it is done.
  griddep_launch_dependents();
  griddep_wait();

  const int hb = p.bn >> 1;                             // token rows per CTA
  if (warp == 0) {
    // ------------------------------------------------------------------------------------------------------ TMA: tokens
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int unit = first; ok && unit < units; unit += stride) {
        const W4Unit u = w4_unit(p, unit);
        const int b0 = u.tn * p.bn + (int)rank * hb;
        for (int st = u.s0; st < u.s1; ++st) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, status, MP_DEV_TIMEOUT_PRODUCER)) { ok = false; break; }
          if (rank == 0) mbar_arrive_expect_tx(full_bar(s), (uint32_t)(2 * hb * 256));
          pair_load(smem_base + (uint32_t)s * (uint32_t)p.stage_bytes + kW4ABytes, tokens, mapa_shared(full_bar(s), 0), 0, p.b_wide, hb, b0, st * 2, 2);
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
    // The whole warp walks the loop and one elected lane issues: the operands of the instructions are then uniform values,
    // which the compiler keeps where the instruction takes them from; a loop inside one lane's branch moves every descriptor
    // there first (46 cycles per instruction).
    if (rank == 0) {
      int s = 0;
      uint32_t ph = 0, ui = 0;
      bool ok = true;
      const uint32_t idesc = umma_idesc(1u, BF16 ? 1u : 0u, kPairRows, (uint32_t)p.bn) | ((uint32_t)p.grad << 15);
      const uint64_t a_base = p.grad ? umma_smem_desc_mn(smem_base, 16384u) : umma_smem_desc_sw128(smem_base);
      const uint64_t b_base = umma_smem_desc_sw128(smem_base) + (kW4ABytes >> 4);
      const uint32_t stage16 = (uint32_t)p.stage_bytes >> 4;
      // 64 contraction elements further: the next block of K-major lines, or 64 MN-major lines; 16: 32 bytes, or 16 lines
      const uint32_t a_step = p.grad ? 2048u >> 4 : 2u, a_blk = p.grad ? 8192u >> 4 : 16384u >> 4, b_blk = (uint32_t)hb * 128u >> 4;
      for (int unit = first; ok && unit < units; unit += stride, ++ui) {
        const W4Unit u = w4_unit(p, unit);
        const uint32_t buf = ui & 1u, use = ui >> 1;
        if (!wait_all(tempty_bar((int)buf), (use & 1u) ^ 1u, status, MP_DEV_TIMEOUT_MMA_TMEM)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * (uint32_t)kPairMaxBN;
        uint32_t more = 0u;
        for (int st = u.s0; st < u.s1; ++st) {
          if (!wait_all(full_bar(s), ph, status, MP_DEV_TIMEOUT_MMA_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint64_t ad = a_base + (uint64_t)((uint32_t)s * stage16), bd = b_base + (uint64_t)((uint32_t)s * stage16);
          if (elect_one()) {
#pragma unroll
            for (uint32_t kk = 0; kk < 8; ++kk) {
              const uint64_t da = ad + (kk >> 2) * a_blk + (kk & 3u) * a_step, db = bd + (kk >> 2) * b_blk + (kk & 3u) * 2u;
              umma_f16_pair(d_tmem, da, db, idesc, kk > 0 ? 1u : more);
            }
            tc_commit_pair(empty_bar(s));
          }
          __syncwarp();
          more = 1u;
          if (++s == stages) { s = 0; ph ^= 1u; }
        }
        if (ok && elect_one()) tc_commit_pair(tfull_bar((int)buf));
        __syncwarp();
      }
    }
  } else if (warp == 2) {
    // ----------------------------------------- TMA: packed weight, as far ahead as its own ring allows (it comes from HBM)
    if (lane == 0) {
      int rs = 0;
      uint32_t rph = 0;
      bool ok = true;
      for (int unit = first; ok && unit < units; unit += stride) {
        const W4Unit u = w4_unit(p, unit);
        for (int st = u.s0; st < u.s1; st += 2) {
          if (!mbar_wait(rempty_bar(rs), rph ^ 1u, status, MP_DEV_TIMEOUT_PRODUCER)) { ok = false; break; }
          mbar_arrive_expect_tx(rfull_bar(rs), kW4RawBytes);
          const uint32_t dst = raw_base + (uint32_t)rs * kW4RawBytes;
          if (p.grad) {                                  // two tiles of 128 rows, one block wide
            tma_load_2d(dst, &tmW, rfull_bar(rs), (u.tm * 2 + (int)rank) * 64, st * 128);
            tma_load_2d(dst + kW4RawBytes / 2, &tmW, rfull_bar(rs), (u.tm * 2 + (int)rank) * 64, st * 128 + 128);
          } else {                                       // one tile, two blocks wide
            tma_load_2d(dst, &tmW, rfull_bar(rs), st * 64, u.tm * kPairRows + (int)rank * 128);
          }
          if (++rs == raw_slots) { rs = 0; rph ^= 1u; }
        }
      }
      if (!ok) settle_copies();
    }
  } else if (warp >= 8) {
    // -------------------------------------------------------------------------------------------------------- unpacking
    // A lane takes the 16-byte chunk t of two rows 8 apart: eight neighbouring lanes are eight rows, which the swizzles of the
    // packed tile (64 or 128 bytes) and of the operand (128 bytes) all spread over the banks.
    const int group = (warp - 8) >> 3, r0 = ((warp - 8) & 7) * 16 + (lane & 7), t = lane >> 3;
    const uint32_t raw0 = raw_base + (uint32_t)(p.grad ? r0 * 64 + ((t ^ ((r0 >> 1) & 3)) << 4) : r0 * 128 + ((t ^ (r0 & 7)) << 4));
    const uint32_t raw1 = p.grad ? raw0 + kW4RawBytes / 2 : raw0 ^ 64u;              // second step of the turn
    const uint32_t rows8 = p.grad ? 512u : 1024u;                                    // eight rows further
    const uint32_t even_at = smem_base + (uint32_t)(r0 * 128 + ((t ^ (r0 & 7)) << 4)), odd_at = even_at ^ 64u;   // runs 0, 2 and 1, 3
    const uint32_t magic = w4_magic<BF16>();
    const W4Weight& w = p.w;
    constexpr int R = FINE ? 4 : 1;                     // groups that a block of a row meets
    uint32_t sz[2][R];                                  // scale | zero << 16
    // Scales and zeros of the lane's two rows, a step ahead of their use: from the table, or (one group per block and row) from
    // where they lie.  Weights that do not exist (rows past N, runs past K) get scale 0: they are zero whatever their bits say.
    const auto fetch = [&](int tm, int st) {
      const int blk = p.grad ? tm * 2 + (int)rank : st;
      const int row = (p.grad ? st * 128 : tm * kPairRows + (int)rank * 128) + r0;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int run = blk * 4 + i, group_at = run >> w.shift;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool real = row + 8 * h < w.N && run * 32 < w.K;
          if (FINE || p.table != nullptr) {
            sz[h][i] = real ? __ldg(p.table + (long long)group_at * p.ld_table + row + 8 * h) : 8u << 16;
          } else {
            const long long at = (long long)(row + 8 * h) * w.groups + group_at;
            const uint32_t z = real && w.zero != nullptr ? (uint32_t)__ldg(w.zero + at) : 8u;
            sz[h][i] = (real ? (uint32_t)__ldg(w.scale + at) : 0u) | z << 16;
          }
        }
      }
    };
    // This CTA's turns (two steps, or the odd last one of a unit), dealt to the two groups alternately across the units.
    struct Turn { int unit, st, s1, tm; };
    const auto open_unit = [&](Turn& x) {
      if (x.unit < units) { const W4Unit u = w4_unit(p, x.unit); x.st = u.s0; x.s1 = u.s1; x.tm = u.tm; }
    };
    // To the next turn; returns the steps of this one that a stage counter has to pass over.
    const auto advance = [&](Turn& x) {
      const int n = min(2, x.s1 - x.st);
      x.st += 2;
      if (x.st >= x.s1) { x.unit += stride; open_unit(x); }
      return n;
    };
    int s = 0, rs = 0;
    uint32_t ph = 0, rph = 0;
    const auto pass = [&](int n) {                       // n stages and one slot further
      s += n;
      if (s >= stages) { s -= stages; ph ^= 1u; }
      if (++rs == raw_slots) { rs = 0; rph ^= 1u; }
    };
    Turn cur{first, 0, 0, 0};
    open_unit(cur);
    if (group == 1 && cur.unit < units) pass(advance(cur));
    if (cur.unit < units) fetch(cur.tm, cur.st);
    bool ok = true;
    while (ok && cur.unit < units) {
      Turn nxt = cur;
      const int mine = advance(nxt);
      int theirs = 0;
      if (nxt.unit < units) theirs = advance(nxt);
      if (!wait_all(rfull_bar(rs), rph, status, MP_DEV_TIMEOUT_MMA_FULL)) break;
      const uint32_t slot = (uint32_t)rs * kW4RawBytes;
      int sh = s;
      uint32_t phh = ph;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (half >= mine) break;
        uint32_t scale[2][R];
        W4Zero zero[2][R];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < R; ++i) { scale[h][i] = (sz[h][i] & 0xffffu) * 0x10001u; zero[h][i] = w4_zero<BF16>(sz[h][i] >> 16); }
        if (half + 1 < mine) fetch(cur.tm, cur.st + 1);
        else if (nxt.unit < units) fetch(nxt.tm, nxt.st);
        const uint32_t from = (half == 0 ? raw0 : raw1) + slot;
        const uint4 q0 = ld_smem_v4<0>(from), q1 = ld_smem_v4<0>(from + rows8);
        if (half + 1 == mine) {
          __syncwarp();
          if (lane == 0) mbar_arrive(rempty_bar(rs));
        }
        if (!wait_all(empty_bar(sh), phh ^ 1u, status, MP_DEV_TIMEOUT_PRODUCER)) { ok = false; break; }
        const uint32_t ev = even_at + (uint32_t)sh * (uint32_t)p.stage_bytes, od = odd_at + (uint32_t)sh * (uint32_t)p.stage_bytes;
        // the weight in the operand type: one rounding of the exact product (q - zero) * scale
        st_smem_v4<0>(ev, w4_weights<BF16>(q0.x, magic, zero[0][0], scale[0][0]));
        st_smem_v4<0>(od, w4_weights<BF16>(q0.y, magic, zero[0][1 % R], scale[0][1 % R]));
        st_smem_v4<16384>(ev, w4_weights<BF16>(q0.z, magic, zero[0][2 % R], scale[0][2 % R]));
        st_smem_v4<16384>(od, w4_weights<BF16>(q0.w, magic, zero[0][3 % R], scale[0][3 % R]));
        st_smem_v4<1024>(ev, w4_weights<BF16>(q1.x, magic, zero[1][0], scale[1][0]));
        st_smem_v4<1024>(od, w4_weights<BF16>(q1.y, magic, zero[1][1 % R], scale[1][1 % R]));
        st_smem_v4<17408>(ev, w4_weights<BF16>(q1.z, magic, zero[1][2 % R], scale[1][2 % R]));
        st_smem_v4<17408>(od, w4_weights<BF16>(q1.w, magic, zero[1][3 % R], scale[1][3 % R]));
        fence_async_smem();                              // the tensor cores read through the async proxy
        __syncwarp();
        if (lane == 0) mbar_arrive_pair(mapa_shared(full_bar(sh), 0));
        if (++sh == stages) { sh = 0; phh ^= 1u; }
      }
      pass(mine);
      if (theirs) pass(theirs);
      cur = nxt;
    }
  } else if (warp >= 4) {
    // --------------------------------------------------------------------------------------------------------- epilogue
    const int quad = warp & 3;
    uint32_t ui = 0;
    for (int unit = first; unit < units; unit += stride, ++ui) {
      const W4Unit u = w4_unit(p, unit);
      const uint32_t buf = ui & 1u, use = ui >> 1;
      const int row = u.tm * kPairRows + (int)rank * 128 + quad * 32 + lane;
      const bool live = row < p.rows;
      const float bias = live && p.bias != nullptr ? from16<BF16>(p.bias[row]) : 0.0f;
      if (!wait_all(tfull_bar((int)buf), use & 1u, status, MP_DEV_TIMEOUT_EPILOGUE)) break;
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
