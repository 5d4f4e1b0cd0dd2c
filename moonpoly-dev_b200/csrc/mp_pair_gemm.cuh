// Persistent tcgen05 GEMM on CTA pairs (cta_group::2):   D[rows x cols] = A * B^T over a common contraction index.
//
// A pair of CTAs (a cluster of two) owns a 256 x bn tile: CTA r of the pair holds rows 128 r ... 128 r + 127 of the tile
// in its TMEM, loads its own 128 rows of A and its own half of the bn rows of B, and the tensor cores of both SMs read
// both halves of B.  Per 64 contraction elements a CTA thus ingests 16 KB + bn / 2 * 128 bytes for 128 * bn * 64 FMAs --
// the operand traffic of a 256 x bn single-CTA tile -- while a tile's accumulator needs only bn TMEM columns, so two
// accumulators fit and the drain of one tile overlaps the main loop of the next.
//
// Either operand may be stored with the contraction index contiguous ("K-major", as the RCC contract gives) or with its
// own row index contiguous ("MN-major": what the gradients need, dX = dY * W and dW = dY^T * X read W, dY and X as they
// lie, without transposed copies).  Both forms are TMA boxes of 128 contiguous bytes per line, 128-byte swizzled.
//
// Roles per CTA: warp 0 = TMA producer, warp 1 = MMA issuer (rank 0 of the pair only) and TMEM owner, warps 4..11 =
// epilogue (TMEM lane quadrant = warp % 4, two warps per quadrant taking the two halves of the columns).
// Barriers: full[s] lives in rank 0 and counts the bytes of both CTAs; empty[s] and tfull[b] exist in both CTAs and are
// signalled by multicast commits; tempty[b] lives in rank 0 and takes the arrivals of the 16 epilogue warps of the pair.
// No TMA load uses cluster multicast.  Every wait is bounded (mbar_wait), as in mp_umma_gemm.cuh.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mp_host.h"
#include "mp_ptx.cuh"

namespace mp {

constexpr int kPairRows = 256;               // rows of D per tile
constexpr int kPairMaxBN = 256;
constexpr int kPairThreads = 384;             // warp 2 of PAIR_STORE(_LONG) posts units; it and warp 3 fill the first warpgroup up
constexpr int kPairMaxStages = 8;
constexpr int kPairSmem = 232448;            // 227 KB opt-in limit per CTA
constexpr int kPairBarBytes = 512;           // behind the stages: barriers, unit box, TMEM address, 8 floats
constexpr int kPairBox = 8, kPairAhead = 2;  // slots of the unit box, and units that it holds ahead of the slowest of its readers

// PAIR_STORE_LONG: PAIR_STORE for contractions of more than kPairStoreChunk blocks, which no single accumulator sums.
enum { PAIR_STORE = 0, PAIR_LSE = 1, PAIR_DLOGITS = 2, PAIR_STORE_LONG = 3 };

// One GEMM of a launch.  A launch may hold two (they share the persistent grid, so the partly empty last wave of one is
// filled by the other).
struct PairProblem {
  int rows, cols, kblocks;       // extents of D, 64-element blocks of the contraction
  int tiles_m, tiles_n, bn;
  int a_mn, b_mn;                // 1: MN-major operand
  int a_rows;                    // rows of A that a CTA loads: 128, or fewer (a multiple of 8) where D has fewer altogether; the
                                 // rest of the tile is whatever lies behind them, and so are its sums, which nobody stores
  int a_wide, b_wide;            // whole blocks of 64 along the operand's lines (see OperandMaps)
  int group_m;                   // raster: tiles are walked in groups of `group_m` row tiles
  int tile0;                     // index of the problem's first unit in the launch
  int split, kb_per_split;       // PAIR_STORE(_LONG): the contraction in `split` slices of kb_per_split blocks, a unit each
  // PAIR_STORE(_LONG): out16 = scale * (acc (+ acc32)), or acc32[slice] (+)= acc when out16 is null
  void* out16;
  float* acc32;
  long long ld_out;              // row stride of out16 in elements
  long long ld_acc, acc_slice;   // row stride of acc32, and elements from slice to slice
  int add_acc32;                 // 1: acc32 holds earlier contributions
};

struct PairParams {
  int num_problems;
  PairProblem prob[2];
  int total_tiles;               // units of the launch
  unsigned* next_unit;           // counter that hands out the units of PAIR_STORE(_LONG); PAIR_DLOGITS, which goes before, clears it
  int stages, stage_bytes;
  int kc;                        // 64-element blocks of the contraction per stage (1 or 2)
  int bf16;                      // operand and output type: 1 = bf16, 0 = fp16
  const float* scale;            // PAIR_STORE(_LONG): device scalar
  int* status;
  // PAIR_LSE / PAIR_DLOGITS (the columns of D are vocabulary entries col0 ... col0 + cols - 1)
  const void* target; int target64;
  long long ignore_index;
  int col0;
  float2* partial;               // PAIR_LSE: [2 * tiles_n][rows] (max, sum of exp(z - max))
  float* target_logit;           // PAIR_LSE: [rows]
  const float* lse;              // PAIR_DLOGITS
  const float* grad_loss;        // PAIR_DLOGITS: [rows], the gradient with respect to the rows' losses
  int vocab;                     // PAIR_DLOGITS: targets are below it
  float* scale_out;              // PAIR_DLOGITS: what the products of d are to be multiplied by
  uint16_t* dlogits; long long ld_dl;
};

// ------------------------------------------------------------------------------------------------- PTX for CTA pairs
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst_smem, const CUtensorMap* tm, uint32_t cluster_bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst_smem), "l"(reinterpret_cast<uint64_t>(tm)), "r"(cluster_bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst_smem, const CUtensorMap* tm, uint32_t cluster_bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst_smem), "l"(reinterpret_cast<uint64_t>(tm)), "r"(cluster_bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// Arrive on a barrier of either CTA of the pair, default semantics: what is handed over is read or written by the tensor
// cores and TMA only, and is ordered by tcgen05 fences or a proxy fence before the arrival.  The cluster-scope release that
// plain memory would need costs a fence each time.
__device__ __forceinline__ void mbar_arrive_pair(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// Arrive on the barrier at this shared-memory offset in both CTAs once all MMAs issued so far have completed.
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void umma_f16_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// MN-major tile, 128-byte swizzle: lines of 64 row indices (128 bytes), one line per contraction index, 8 lines per
// swizzle atom (1024 bytes apart); `block_bytes` separates consecutive blocks of 64 row indices.
__device__ __forceinline__ uint64_t umma_smem_desc_mn(uint32_t saddr, uint32_t block_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3ffffu) >> 4);
  d |= static_cast<uint64_t>(block_bytes >> 4) << 16;         // leading byte offset: next 64 row indices
  d |= static_cast<uint64_t>(1024 >> 4) << 32;                // stride byte offset: next 8 contraction indices
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// Registers per thread of a warpgroup from here on.  The launch has 384 x 168; 128 x 88 + 256 x 208 is just that.
__device__ __forceinline__ void regs_fewer_88() { asm volatile("setmaxnreg.dec.sync.aligned.u32 88;"); }
__device__ __forceinline__ void regs_more_208() { asm volatile("setmaxnreg.inc.sync.aligned.u32 208;"); }
// mbar_wait by a whole warp, with one answer for it: where a wait gives up, no lane may go on to the warp's next aligned instruction
// or __syncwarp without the others.
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, int* status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code)) != 0;
}
__device__ __forceinline__ float exp2_approx(float x) {        // 2^x, 2 ulp, subnormal results flushed to zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// After an error: give copies already under way (their barrier may be the peer's) ample time to land.
__device__ __forceinline__ void settle_copies() {
  const unsigned long long t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 5000000ull) {}
}

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ uint32_t pack16(float a, float b, int bf16) {
  if (bf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A warp's block of 32 rows x 64 columns of 16-bit outputs, one row per lane in w, to `o` (its first element; rows `ld`
// elements apart; `rows` x `cols` of it exist).  By way of 4 KB of shared memory, so that eight lanes write 128 contiguous
// bytes of a row.  Lanes that wrote their own rows, 16 bytes each, left a part of a sector in 32 rows behind every instruction
// (both gradients, us: 128 x 32768 x 4096 260 -> 218, 2048 x 32768 x 1023, where rows miss 16 bytes, 538 -> 347,
// 10 x 21273 x 3280 148 -> 135).  Blocks that end inside the 64 columns take the same path while whole 16 bytes of them are
// left (2 x 9964 x 1744: 47 -> 41).
__device__ __forceinline__ void store_rows64(uint32_t stage, uint16_t* o, long long ld, int rows, int cols, const uint32_t (&w)[32], int lane) {
  __syncwarp();                                          // the previous block has been read
#pragma unroll
  for (int c = 0; c < 8; ++c)
    st_smem_v4(stage + (uint32_t)(lane * 128 + ((c ^ (lane & 7)) << 4)), make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
  __syncwarp();
  if ((cols >= 64 || cols % 8 == 0) && ((reinterpret_cast<uintptr_t>(o) | (uintptr_t)(ld * 2)) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * 4 + (lane >> 3), c = lane & 7;
      uint4 v;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                   : "r"(stage + (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4))) : "memory");
      if (r < rows && c * 8 < cols) *reinterpret_cast<uint4*>(o + r * ld + c * 8) = v;
    }
  } else {                                               // rows that miss 16 bytes
    const bool c0 = lane < cols, c1 = lane + 32 < cols;
    const uint32_t in = stage + (uint32_t)(lane & 7) * 2;
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
      uint16_t v0, v1;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v0) : "r"(in + (uint32_t)(r * 128 + (((lane >> 3) ^ (r & 7)) << 4))) : "memory");
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v1) : "r"(in + (uint32_t)(r * 128 + (((4 + (lane >> 3)) ^ (r & 7)) << 4))) : "memory");
      if (c0 && r < rows) o[r * ld + lane] = v0;
      if (c1 && r < rows) o[r * ld + lane + 32] = v1;
    }
  }
}
constexpr int kPairStoreBytes = 8 * 4096;                // of the eight epilogue warps

// The tensor maps of an operand.  `wide` is 3-D and one box brings 256 contiguous bytes per line, two blocks of 64 (1.07 times
// as fast a main loop as 128-byte boxes); it covers whole blocks only.  `narrow` covers the lines to their last element and is
// there for the boxes that would reach past the last whole block.
struct alignas(64) OperandMaps { CUtensorMap wide, narrow; };
struct PairMaps { OperandMaps a[2], b[2]; };          // of the launch's problems

// Maps of a row-major 16-bit matrix of `rows` lines of `inner` elements, `ld` apart, for boxes of `box_lines` lines and
// `box_blocks` blocks of 64 elements.
inline int operand_maps(OperandMaps* m, const void* ptr, long long inner, long long rows, long long ld, int box_lines, int box_blocks, int* whole) {
  *whole = inner % 64 == 0 ? 1 << 24 : (int)(inner / 64);      // a line of whole blocks: the fill beyond it does the rest
  if (inner >= 64) {
    if (int rc = host_tmap_blocks(&m->wide, ptr, inner / 64 * 64, rows, ld * 2, box_lines, box_blocks)) return rc;
  }
  if (inner % 64 != 0) {
    if (int rc = host_tmap(&m->narrow, kTmap16, ptr, inner, rows, ld * 2, 64, box_lines, 128)) return rc;
  } else {
    m->narrow = m->wide;
  }
  if (inner < 64) m->wide = m->narrow;                         // never loaded through, but a valid map
  return 0;
}

// One stage of one operand: `rows` row indices from r0, contraction blocks kb ... kb + kc - 1.  K-major: [block][row][128 B];
// MN-major: [64 row indices][kc * 64 contraction indices][128 B].  `blocks` whole blocks of 64 along the lines may be read
// through the wide map.  Blocks past the end of the contraction are filled with zeros and count their bytes like the others.
__device__ __forceinline__ void pair_load(uint32_t dst, const OperandMaps& maps, uint32_t bar, int mn, int blocks, int rows, int r0, int kb, int kc) {
  if (mn) {
    if (r0 + rows <= blocks * 64) tma_load_3d_pair(dst, &maps.wide, bar, 0, kb * 64, r0 >> 6);
    else for (int j = 0; j < rows; j += 64) tma_load_2d_pair(dst + (uint32_t)(j * kc * 128), &maps.narrow, bar, r0 + j, kb * 64);
  } else if (kb + kc <= blocks) {
    tma_load_3d_pair(dst, &maps.wide, bar, 0, r0, kb);
  } else {
    for (int c = 0; c < kc; ++c) tma_load_2d_pair(dst + (uint32_t)(c * rows * 128), &maps.narrow, bar, (kb + c) * 64, r0);
  }
}

struct PairUnit { int prob, tm, tn, slice, kb0, kb1; };

__host__ __device__ __forceinline__ PairUnit pair_unit(const PairParams& p, int unit) {
  PairUnit u;
  u.prob = (p.num_problems == 2 && unit >= p.prob[1].tile0) ? 1 : 0;
  const PairProblem& q = p.prob[u.prob];
  int t = unit - q.tile0;
  u.slice = 0;
  u.kb0 = 0;
  u.kb1 = q.kblocks;
  if (q.split > 1) {                                     // slice by slice: neighbours share the operands of a slice
    const int tiles = q.tiles_m * q.tiles_n;
    u.slice = t / tiles;
    t -= u.slice * tiles;
    u.kb0 = u.slice * q.kb_per_split;
    u.kb1 = u.kb0 + q.kb_per_split < q.kblocks ? u.kb0 + q.kb_per_split : q.kblocks;
  }
  const int group = q.group_m * q.tiles_n;
  const int g = t / group, first = g * q.group_m;
  const int height = q.tiles_m - first < q.group_m ? q.tiles_m - first : q.group_m;
  const int in = t - g * group;
  u.tn = in / height;
  u.tm = first + (in - u.tn * height);
  return u;
}

// Where the roles of a CTA get their units from.  Static: pair, pair + pairs, ...  Dynamic (units of different lengths):
// the first unit is the pair's own number, further ones come from a counter in global memory; warp 2 of rank 0 fetches them
// and posts them in a box in the shared memory of both CTAs.  The producers and the MMA issuer hand a unit back when they
// read it.  The epilogue warps do not: an arrival in the other CTA would wait for the stores behind them (128 x 32768 x 4096,
// both gradients: 218 us instead of 204).  The box has kPairBox slots for that: a unit is posted when the one kPairAhead
// before it has been handed back; the MMA issuer has then seen the accumulator free that the third unit before that one
// filled, and kPairAhead + 3 <= kPairBox.  Taking 3 or 4 units ahead is no faster, 1 is slower by 5 %.
// Which pair computes a unit has no influence on its result.
template <bool DYNAMIC>
struct PairUnits {
  const PairParams& p;
  uint32_t box, bars;            // slots (4 bytes each) and barriers (box_full[kPairBox], box_empty[kPairBox], 8 bytes each)
  int unit, step;
  uint32_t n = 0;
  __device__ PairUnits(const PairParams& p_, uint32_t box_, uint32_t bars_, int pair, int pairs) : p(p_), box(box_), bars(bars_), unit(pair - pairs), step(pairs) {}
  // The next unit, or -1.  Called by one lane.
  __device__ __forceinline__ int next(bool hands_back = true) {
    if constexpr (!DYNAMIC) {
      unit += step;
      return unit < p.total_tiles ? unit : -1;
    } else {
      const uint32_t slot = n % kPairBox, ph = n / kPairBox & 1u;
      ++n;
      if (!mbar_wait_cluster(bars + 8u * slot, ph, p.status, MP_DEV_TIMEOUT_CLUSTER)) return -1;
      int v;
      asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v) : "r"(box + 4u * slot) : "memory");
      if (hands_back) mbar_arrive_cluster(mapa_shared(bars + 8u * (kPairBox + slot), 0));
      return v < p.total_tiles ? v : -1;
    }
  }
  // Warp 2 of rank 0, one lane: posts units until the roles have been told that there are none left.
  __device__ __forceinline__ void post(int pair, int pairs) {
    for (uint32_t i = 0;; ++i) {
      const uint32_t slot = i % kPairBox, back = i - (uint32_t)kPairAhead;
      if (i >= (uint32_t)kPairAhead &&
          !mbar_wait_cluster(bars + 8u * (kPairBox + back % kPairBox), back / kPairBox & 1u, p.status, MP_DEV_TIMEOUT_CLUSTER)) return;
      const int v = i == 0 ? pair : (int)atomicAdd(p.next_unit, 1u) + pairs;
      for (uint32_t r = 0; r < 2; ++r) {
        asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(mapa_shared(box + 4u * slot, r)), "r"(v) : "memory");
        mbar_arrive_cluster(mapa_shared(bars + 8u * slot, r));
      }
      if (v >= p.total_tiles) return;
    }
  }
};

// ------------------------------------------------------------------------------------------------------ the epilogues
// The tensor cores drop the bits that an addition shifts out, always towards zero, so a long contraction pulls every logit to
// zero, which the mean over a vocabulary does not average away.  The contraction therefore comes in chunks of kPairChunk
// blocks, each in an accumulator of its own, and the chunks are added here, rounded to nearest, while the other accumulator is
// being filled: at H = 4096 and logits of deviation 2, lse (11 in size) is off by 4e-6 on average instead of 1.7e-5, at H = 16384 by
// 4e-6 instead of 6.8e-5.  The forward pass and the gradients' logits take the same chunks and get the same bits: at the target d
// is exp(z - lse) - 1, and of a nearly certain row nothing else is left.
constexpr int kPairChunk = 16;               // blocks of 64 contraction elements per accumulator
// The gradients, rounded to 16 bits in the end, take longer chunks: 512 additions leave a sum short by 2^-16 of itself at most, 1/32 of
// fp16's half step; the 8192 of 131072 vocabulary entries left 1.3e-4.  The chunks of PAIR_STORE_LONG are summed in registers, and
// tiles with little to multiply then leave more slowly: loss and both gradients of 128 x 32768 x 4096 take 284 us with it and 271
// with PAIR_STORE, whose slices of one chunk are written in 32 bits and joined.  At 2048 x 32768 x 1024 it costs 1 %.
constexpr int kPairStoreChunk = 128;
template <int EPI> struct PairEpi {
  static constexpr bool kStores = EPI == PAIR_STORE || EPI == PAIR_STORE_LONG, kSums = EPI != PAIR_STORE;
  static constexpr int kChunk = kStores ? kPairStoreChunk : kPairChunk;      // PAIR_STORE never has more than one
};

// z += this warp's half (128 columns) of the accumulator, one row per lane; t_addr: its first column.
__device__ __forceinline__ void pair_add_chunk(float (&z)[128], uint32_t t_addr) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t v[32];
    __syncwarp();
    tmem_ld_x32(t_addr + 32u * c, v);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 32; ++j) z[32 * c + j] += __uint_as_float(v[j]);
  }
}

// Softmax statistics of this warp's half of a 256-column tile, one row per lane.
// The maximum is taken first and z - max is formed before the multiplication by log2(e), so that the sum is exact to a
// few units in the last place whatever the logits' size.  An infinite maximum is replaced by 0 (exp then gives 0 or
// infinity as the definition does); NaN passes through the sum.  The 128 terms are added in pairs: beside a nearly certain entry's 1,
// terms below 2^-24 would vanish one by one (2000 entries of 4e-8: the loss is off by 2e-7 instead of 1.7e-6).
__device__ __forceinline__ void pair_epilogue_lse(const PairParams& p, const PairProblem& q, float (&z)[128], int row, int c_begin,
                                                  int tn, int half, int ncols) {
  const bool live = row < q.rows;
  long long target = -1;
  if (live) {
    const long long t = p.target64 ? reinterpret_cast<const long long*>(p.target)[row] : reinterpret_cast<const int*>(p.target)[row];
    if (t != p.ignore_index) target = t - c_begin;                       // column inside this warp's half, if any
  }
  float m = -INFINITY;
  const bool full = ncols >= 128;
#pragma unroll
  for (int j = 0; j < 128; ++j) if (full || j < ncols) m = fmaxf(m, z[j]);
  if (target >= 0 && target < ncols && target < 128) {
    float t = 0.0f;
#pragma unroll
    for (int j = 0; j < 128; ++j) if (target == j) t = z[j];
    p.target_logit[row] = t;
  }
  const float base = isinf(m) ? 0.0f : m;
#pragma unroll
  for (int j = 0; j < 128; ++j) z[j] = full || j < ncols ? exp2_approx((z[j] - base) * kLog2e) : 0.0f;
#pragma unroll
  for (int w = 64; w; w >>= 1) {
#pragma unroll
    for (int j = 0; j < w; ++j) z[j] += z[j + w];
  }
  // a half without columns keeps (-inf, 0)
  if (live) p.partial[(size_t)(2 * tn + half) * q.rows + row] = make_float2(m, z[0]);
}

// The largest finite |grad_loss| of the rows that have a loss (1 if there is none), by the eight epilogue warps while the
// first tile is being multiplied; `slots` are 8 floats of shared memory.
__device__ __forceinline__ float pair_grad_max(const PairParams& p, int rows, float* slots) {
  const int e = (int)threadIdx.x - 128;
  float g = 0.0f;
  for (int i = e; i < rows; i += 256) {
    const long long t = p.target64 ? reinterpret_cast<const long long*>(p.target)[i] : reinterpret_cast<const int*>(p.target)[i];
    const float a = fabsf(p.grad_loss[i]);
    if (t != p.ignore_index && a < INFINITY) g = fmaxf(g, a);          // infinities and NaN go through as they are
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
  if ((e & 31) == 0) slots[e >> 5] = g;
  asm volatile("bar.sync 1, 256;" ::: "memory");
  g = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) g = fmaxf(g, slots[i]);
  return g == 0.0f ? 1.0f : g;
}

// d = grad_loss[row] * (softmax - onehot), rounded once to the operand type and parked for the two gradient products.  The
// largest |grad_loss| is divided out (a mean over the tokens then rounds exactly: the factors are 1) and, for fp16, replaced
// by 2^15: a probability of 2e-9 is still a normal fp16 number beside a one.  The products are multiplied by *scale_out.
__device__ __forceinline__ void pair_epilogue_dlogits(const PairParams& p, const PairProblem& q, const float (&z)[128], int row, int c_begin,
                                                      int ncols, float grad_max, uint32_t stage) {
  const bool live = row < q.rows;
  long long target = -1;
  float lse = 0.0f, coef = 0.0f;
  bool kept = false;
  if (live) {
    const long long t = p.target64 ? reinterpret_cast<const long long*>(p.target)[row] : reinterpret_cast<const int*>(p.target)[row];
    kept = t != p.ignore_index;
    target = t - p.col0 - c_begin;
    lse = p.lse[row];
    coef = t < 0 || t >= p.vocab ? NAN : p.grad_loss[row] / grad_max * (p.bf16 ? 1.0f : 32768.0f);
  }
  const int lane = row & 31, row0 = row - lane;
  uint16_t* o = p.dlogits + (long long)row0 * p.ld_dl + c_begin;
#pragma unroll
  for (int c0 = 0; c0 < 128; c0 += 64) {
    uint32_t w[32];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int c1 = c0 + 32 * part;
      float d[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) d[j] = kept ? coef * exp2_approx((z[c1 + j] - lse) * kLog2e) : 0.0f;
      if (kept && target >= c1 && target < c1 + 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (target == c1 + j) d[j] = coef * (exp2_approx((z[c1 + j] - lse) * kLog2e) - 1.0f);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) w[16 * part + j] = pack16(d[2 * j], d[2 * j + 1], p.bf16);
    }
    if (c0 < ncols) store_rows64(stage, o + c0, p.ld_dl, q.rows - row0, ncols - c0, w, lane);
  }
}

// z: the unit's sums where it has several chunks (SUMS); the only chunk is read from t_addr.
template <bool SUMS>
__device__ __forceinline__ void pair_epilogue_store(const PairParams& p, const PairProblem& q, uint32_t t_addr, const float (&z)[128], int row,
                                                    int c_begin, int ncols, int slice, float scale, uint32_t stage) {
  const bool live = row < q.rows;
  const int lane = row & 31, row0 = row - lane;
  constexpr int kUnroll = SUMS ? 2 : 1;                    // z is indexed
#pragma unroll kUnroll
  for (int c0 = 0; c0 < 128; c0 += 64) {
    uint32_t w[32];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int c1 = c0 + 32 * part;
      float v[32];
      if constexpr (SUMS) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = z[c1 + j];
      } else {
        uint32_t r[32];
        __syncwarp();
        tmem_ld_x32(t_addr + (uint32_t)c1, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
      }
      float* a = q.acc32 + (long long)slice * q.acc_slice + (long long)row * q.ld_acc + c_begin + c1;
      const bool mine = live && c1 < ncols;                // ld_acc is a multiple of 32: rows of the scratch are padded
      if (q.add_acc32 && mine) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 t = reinterpret_cast<const float4*>(a)[j];
          v[4 * j] += t.x; v[4 * j + 1] += t.y; v[4 * j + 2] += t.z; v[4 * j + 3] += t.w;
        }
      }
      if (q.out16 != nullptr) {
#pragma unroll
        for (int j = 0; j < 16; ++j) w[16 * part + j] = pack16(v[2 * j] * scale, v[2 * j + 1] * scale, p.bf16);
      } else if (mine) {
#pragma unroll
        for (int j = 0; j < 8; ++j) reinterpret_cast<float4*>(a)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      }
    }
    if (q.out16 != nullptr && c0 < ncols)
      store_rows64(stage, reinterpret_cast<uint16_t*>(q.out16) + (long long)row0 * q.ld_out + c_begin + c0, q.ld_out, q.rows - row0, ncols - c0, w, lane);
  }
}

// ---------------------------------------------------------------------------------------------------------- the kernel
template <int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
pair_gemm_kernel(const __grid_constant__ PairMaps maps, const PairParams p) {
  extern __shared__ uint8_t smem_raw[];
  // both CTAs of the pair see the same dynamic shared-memory offset, so the rounding agrees
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_base = smem_u32(smem);
  const int stages = p.stages;
  const uint32_t bar_base = smem_base + (uint32_t)stages * (uint32_t)p.stage_bytes;
  auto full_bar = [&](int s) { return bar_base + 8u * (uint32_t)s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (uint32_t)(stages + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (uint32_t)(2 * stages + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (uint32_t)(2 * stages + 2 + b); };
  const uint32_t unit_bars = bar_base + 8u * (uint32_t)(2 * stages + 4), unit_box = unit_bars + 16u * kPairBox;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + (size_t)stages * p.stage_bytes + 8 * (2 * stages + 4) + 20 * kPairBox);
  constexpr bool DYNAMIC = PairEpi<EPI>::kStores, SUMS = PairEpi<EPI>::kSums;
  constexpr int kChunk = PairEpi<EPI>::kChunk;

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
  int* status = p.status;
  PairUnits<DYNAMIC> units(p, unit_box, unit_bars, pair, pairs);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(tfull_bar(b), 1); mbar_init(tempty_bar(b), 16); }
    for (uint32_t b = 0; b < (uint32_t)kPairBox; ++b) {
      mbar_init(unit_bars + 8u * b, 1);
      mbar_init(unit_bars + 8u * (uint32_t)(kPairBox + b), 3);           // two producers and the MMA issuer
    }
    mbar_fence_init();
    for (int i = 0; i < p.num_problems; ++i) { tma_prefetch_desc(&maps.a[i].wide); tma_prefetch_desc(&maps.b[i].wide); }
  }
  if (warp == 1) tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  cluster_sync_all();                       // the peer's barriers are initialised, its TMEM is allocated
  // Everything above may overlap the previous kernel of the stream; nothing of it is read or overwritten before it is done.
  griddep_launch_dependents();
  griddep_wait();

  if (warp < 4) {
    if constexpr (SUMS) regs_fewer_88();                 // the epilogue holds 128 sums per thread
    // ------------------------------------------------------------------------------------------ TMA producer (one lane)
    if (warp == 0 && lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int unit; ok && (unit = units.next()) >= 0;) {
        const PairUnit u = pair_unit(p, unit);
        const PairProblem& q = p.prob[u.prob];
        const int hb = q.bn >> 1;
        const int a0 = u.tm * kPairRows + (int)rank * 128, b0 = u.tn * q.bn + (int)rank * hb;
        // A CTA whose share of an operand lies wholly behind its end loads nothing: boxes of zeros take the TMA unit longer
        // than data (a single row of 4096 against 50021: 116 us with them).
        const uint32_t a_bytes = (uint32_t)(p.kc * q.a_rows * 128), b_bytes = (uint32_t)(p.kc * hb * 128);
        const bool has_a = a0 < q.rows, has_b = b0 < q.cols;
        const uint32_t tx = a_bytes * (u.tm * kPairRows + 128 < q.rows ? 2u : 1u) + b_bytes * (u.tn * q.bn + hb < q.cols ? 2u : 1u);   // both CTAs
        for (int kb = u.kb0; kb < u.kb1; kb += p.kc) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, status, MP_DEV_TIMEOUT_PRODUCER)) { ok = false; break; }
          const uint32_t dst = smem_base + (uint32_t)s * (uint32_t)p.stage_bytes;
          if (rank == 0) mbar_arrive_expect_tx(full_bar(s), tx);
          const uint32_t bar = mapa_shared(full_bar(s), 0);
          if (has_a) pair_load(dst, maps.a[u.prob], bar, q.a_mn, q.a_wide, q.a_rows, a0, kb, p.kc);
          if (has_b) pair_load(dst + a_bytes, maps.b[u.prob], bar, q.b_mn, q.b_wide, hb, b0, kb, p.kc);
          if (++s == stages) { s = 0; ph ^= 1u; }
        }
      }
      // every stage handed back: all copies have landed and all commits have reached this CTA's barriers
      for (int i = 0; ok && i < stages; ++i) {
        ok = mbar_wait(empty_bar(s), ph ^ 1u, status, MP_DEV_TIMEOUT_DRAIN);
        if (++s == stages) { s = 0; ph ^= 1u; }
      }
      if (!ok) settle_copies();
    }
    // ---------------------------------------------------------------------------- MMA issuer (one lane of rank 0's warp)
    // The whole warp walks the loop and one elected lane issues: the operands of the instructions are then uniform values,
    // which the compiler keeps where the instruction takes them from; a loop inside one lane's branch moves every descriptor
    // there first (46 cycles per instruction).
    if (warp == 1 && rank == 0) {
      int s = 0;
      uint32_t ph = 0, ui = 0;
      bool ok = true;
      while (ok) {
        int unit;
        if constexpr (DYNAMIC) {
          unit = lane == 0 ? units.next() : 0;
          unit = __shfl_sync(0xffffffffu, unit, 0);
        } else {
          unit = units.next();
        }
        if (unit < 0) break;
        const PairUnit u = pair_unit(p, unit);
        const PairProblem& q = p.prob[u.prob];
        const uint32_t idesc = umma_idesc(1u, p.bf16 ? 1u : 0u, kPairRows, (uint32_t)q.bn) | ((uint32_t)q.a_mn << 15) | ((uint32_t)q.b_mn << 16);
        const uint32_t mn_block = (uint32_t)p.kc * 8192u;
        const uint64_t a_base = q.a_mn ? umma_smem_desc_mn(smem_base, mn_block) : umma_smem_desc_sw128(smem_base);
        const uint64_t b_base = (q.b_mn ? umma_smem_desc_mn(smem_base, mn_block) : umma_smem_desc_sw128(smem_base)) +
                                (uint64_t)((uint32_t)(p.kc * q.a_rows * 128) >> 4);
        // 16 contraction elements further: 32 bytes along a K-major line, or 16 lines of an MN-major tile; 64 further: the
        // next K-major block, or 64 lines
        const uint32_t a_step = q.a_mn ? 2048u >> 4 : 2u, b_step = q.b_mn ? 2048u >> 4 : 2u;
        const uint32_t a_blk = q.a_mn ? 8192u >> 4 : (uint32_t)q.a_rows * 128u >> 4, b_blk = q.b_mn ? 8192u >> 4 : (uint32_t)(q.bn >> 1) * 128u >> 4;
        const uint32_t stage16 = (uint32_t)p.stage_bytes >> 4;
        for (int k0 = u.kb0; ok && k0 < u.kb1; k0 += kChunk, ++ui) {       // a chunk of the contraction per accumulator
          const uint32_t buf = ui & 1u, use = ui >> 1;
          if (!wait_all(tempty_bar((int)buf), (use & 1u) ^ 1u, status, MP_DEV_TIMEOUT_MMA_TMEM)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + buf * (uint32_t)kPairMaxBN;
          const int k1 = min(u.kb1, k0 + kChunk);
          uint32_t more = 0u;
          for (int kb = k0; kb < k1; kb += p.kc) {
            if (!wait_all(full_bar(s), ph, status, MP_DEV_TIMEOUT_MMA_FULL)) { ok = false; break; }
            tc_fence_after();
            uint64_t ad = a_base + (uint64_t)((uint32_t)s * stage16), bd = b_base + (uint64_t)((uint32_t)s * stage16);
            const int nc = min(p.kc, k1 - kb);
            if (elect_one()) {
              for (int c = 0; c < nc; ++c, ad += a_blk, bd += b_blk) {
#pragma unroll
                for (uint32_t kk = 0; kk < 4; ++kk) umma_f16_pair(d_tmem, ad + kk * a_step, bd + kk * b_step, idesc, kk > 0 ? 1u : more);
                more = 1u;
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
    }
    if constexpr (DYNAMIC) {
      if (warp == 2 && lane == 0 && rank == 0) units.post(pair, pairs);
    }
  } else {
    // -------------------------------------------------------------------------------------------------- epilogue warps
    if constexpr (SUMS) regs_more_208();
    const int quad = warp & 3, half = (warp - 4) >> 2;
    uint32_t ui = 0;
    bool ok = true;
    float grad_max = 1.0f;
    const uint32_t stage = bar_base + kPairBarBytes + (uint32_t)(warp - 4) * 4096u;       // of this warp, where outputs are 16 bits (kPairStoreBytes)
    const float scale = DYNAMIC ? *p.scale : 1.0f;
    if constexpr (EPI == PAIR_DLOGITS) {
      grad_max = pair_grad_max(p, p.prob[0].rows, reinterpret_cast<float*>(smem + (size_t)stages * p.stage_bytes + 8 * (2 * stages + 4) + 20 * kPairBox + 8));
      if (blockIdx.x == 0 && threadIdx.x == 128) {
        *p.scale_out = grad_max / (p.bf16 ? 1.0f : 32768.0f);
        *p.next_unit = 0u;                               // of the products' launch
      }
    }
    while (ok) {
      int unit = 0;
      if constexpr (DYNAMIC) {
        if (lane == 0) unit = units.next(false);
        unit = __shfl_sync(0xffffffffu, unit, 0);
      } else {
        unit = units.next();
      }
      if (unit < 0) break;
      const PairUnit u = pair_unit(p, unit);
      const PairProblem& q = p.prob[u.prob];
      const int half_cols = q.bn >> 1;
      const int row = u.tm * kPairRows + (int)rank * 128 + quad * 32 + lane;
      const int c_begin = u.tn * q.bn + half * half_cols;                // first column of this warp's half
      const int ncols = min(half_cols, q.cols - c_begin);                // may be <= 0 in the last column tile
      const uint32_t t_half = tmem_base + (uint32_t)(half * half_cols) + ((uint32_t)(quad * 32) << 16);
      float z[128];
      if constexpr (SUMS) {
#pragma unroll
        for (int j = 0; j < 128; ++j) z[j] = 0.0f;
        for (int k0 = u.kb0; ok && k0 < u.kb1; k0 += kChunk, ++ui) {
          const uint32_t buf = ui & 1u, use = ui >> 1;
          if (!wait_all(tfull_bar((int)buf), use & 1u, status, MP_DEV_TIMEOUT_EPILOGUE)) { ok = false; break; }
          tc_fence_after();
          pair_add_chunk(z, t_half + buf * (uint32_t)kPairMaxBN);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_pair(mapa_shared(tempty_bar((int)buf), 0));
        }
        if (!ok) break;
        if constexpr (EPI == PAIR_LSE) pair_epilogue_lse(p, q, z, row, c_begin, u.tn, half, ncols);
        else if constexpr (EPI == PAIR_DLOGITS) pair_epilogue_dlogits(p, q, z, row, c_begin, ncols, grad_max, stage);
        else pair_epilogue_store<true>(p, q, 0u, z, row, c_begin, ncols, u.slice, scale, stage);
      } else {
        const uint32_t buf = ui & 1u, use = ui >> 1;
        if (!wait_all(tfull_bar((int)buf), use & 1u, status, MP_DEV_TIMEOUT_EPILOGUE)) break;
        tc_fence_after();
        pair_epilogue_store<false>(p, q, t_half + buf * (uint32_t)kPairMaxBN, z, row, c_begin, ncols, u.slice, scale, stage);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_pair(mapa_shared(tempty_bar((int)buf), 0));
        ++ui;
      }
    }
  }

  // Neither CTA may leave while the other can still read its shared memory, signal its barriers or use its TMEM.
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

}  // namespace mp
