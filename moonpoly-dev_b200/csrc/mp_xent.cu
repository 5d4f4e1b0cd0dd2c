// Linear with softmax cross entropy (mp_linear_xent, mp_linear_xent_grad): z = X W^T over a vocabulary of V entries,
// loss = logsumexp(z) - z[target], and the gradients of X and W, without ever holding the [M, V] logits.
//
// Forward: one pass of the CTA-pair GEMM whose epilogue reduces every 256 x 256 tile of logits to a maximum and a sum of
// exponentials per row and half tile; a small kernel joins the pieces.
// Gradients: d = g (softmax(z) - onehot), dX = d W, dW = d^T X.  The vocabulary is walked in pieces; a piece's logits are
// computed again, turned into d in the epilogue and parked in 16 bits, and one launch runs both gradient products of the
// piece from there.  dX is summed over the pieces in 32 bits, in the order of the pieces.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/moonpoly_abi.h"
#include "mp_host.h"
#include "mp_pair_gemm.cuh"

namespace {

using namespace mp;

size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

// ---------------------------------------------------------------------------------------------------- small kernels
// What a sum of exp(z - m) is to be multiplied by where the row's maximum is `top`.  Equal maxima, two infinite ones among them, keep
// their sums as they are; an infinite one makes the others vanish, but lets NaN through.
__device__ __forceinline__ float rescale(float m, float top) { return m == top ? 1.0f : exp2_approx((m - top) * kLog2e); }

// loss and logsumexp of every row from the partial (max, sum) pairs; 32 rows x 32 groups of partials per block.
__global__ void __launch_bounds__(1024) xent_join_kernel(const float2* partial, int num, int rows, const float* target_logit,
                                                         const void* target, int target64, long long ignore_index, int vocab,
                                                         float* loss, float* lse) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ float sm[32][33], ss[32][33];
  const int rx = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + rx;
  float m = -INFINITY, s = 0.0f;
  if (row < rows) {
    for (int i = g; i < num; i += 32) {
      const float2 v = partial[(size_t)i * rows + row];
      const float mn = fmaxf(m, v.x);
      s = s * rescale(m, mn) + v.y * rescale(v.x, mn);
      m = mn;
    }
  }
  sm[g][rx] = m;
  ss[g][rx] = s;
  __syncthreads();
  if (g != 0 || row >= rows) return;
  float top = -INFINITY;
  for (int i = 0; i < 32; ++i) top = fmaxf(top, sm[i][rx]);
  float sum[32];                                   // added in pairs, like the terms of a piece
#pragma unroll
  for (int i = 0; i < 32; ++i) sum[i] = ss[i][rx] * rescale(sm[i][rx], top);
#pragma unroll
  for (int w = 16; w; w >>= 1) {
#pragma unroll
    for (int i = 0; i < w; ++i) sum[i] += sum[i + w];
  }
  const float base = isinf(top) ? 0.0f : top;      // the sum is then infinite, zero or NaN itself
  const float logsum = logf(sum[0]);
  lse[row] = base + logsum;
  const long long t = target64 ? reinterpret_cast<const long long*>(target)[row] : reinterpret_cast<const int*>(target)[row];
  if (t == ignore_index) loss[row] = 0.0f;
  else if (t < 0 || t >= vocab) loss[row] = NAN;   // no such entry: loud, and nothing is read out of range
  else loss[row] = logsum + (base - target_logit[row]);   // small losses keep their digits: no large lse is formed
}

// dX = scale * sum of the slices' 32-bit sums, in their order; four columns per thread.
__global__ void __launch_bounds__(256) xent_dx_kernel(const float* acc, int slices, long long slice_words, long long ld_acc, int rows, int cols,
                                                      const float* scale, uint16_t* out, int bf16) {
  griddep_launch_dependents();
  griddep_wait();
  const int quads = (int)(ld_acc >> 2);
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  if (x >= (long long)rows * quads) return;
  const int row = (int)(x / quads), col = (int)(x - (long long)row * quads) * 4;
  const int n = cols - col < 4 ? cols - col : 4;
  if (n <= 0) return;
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < slices; ++i) {
    const float4 a = *reinterpret_cast<const float4*>(acc + i * slice_words + row * ld_acc + col);
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
  }
  const float k = *scale;
  const uint32_t lo = pack16(v[0] * k, v[1] * k, bf16), hi = pack16(v[2] * k, v[3] * k, bf16);
  uint16_t* o = out + (long long)row * cols + col;
  if (n == 4 && (reinterpret_cast<uintptr_t>(o) & 7) == 0) {
    *reinterpret_cast<uint2*>(o) = make_uint2(lo, hi);
  } else {
    const uint16_t w[4] = {(uint16_t)lo, (uint16_t)(lo >> 16), (uint16_t)hi, (uint16_t)(hi >> 16)};
    for (int e = 0; e < n; ++e) o[e] = w[e];
  }
}

// ------------------------------------------------------------------------------------------------------------ problem
// Sizes that follow from the shape alone, so that the workspace query and the call agree.
struct Layout {
  size_t x_copy, w_copy;                  // aligned copies of operands whose rows miss TMA's 16 bytes
  size_t partial, target_logit;           // forward
  size_t scale, dl, acc;                  // gradients (scale: and the unit counter)
  int hp, piece, pieces;
  int max_split;                          // slices that `acc` has room for
  long long ld_acc, ld_dl, acc_slice;
  size_t total;
};

// Vocabulary entries per piece of the gradient.
int xent_piece(int M, int V) {
  const long long rows = std::max<long long>(round_up((size_t)M, 256), 256);
  long long piece = (256ll << 20) / (2 * rows) / 256 * 256;
  piece = std::max<long long>(piece, 4096);
  return (int)std::min<long long>(piece, (long long)round_up((size_t)V, 256));
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

// 64-element contraction blocks per pipeline stage.
constexpr int kStageBlocks = 2;

constexpr int kPairsModel = 74;          // workspace sizes must not depend on the device that is asked

// Slices of the vocabulary in the product dX = d W of one piece.  It has few, long tiles (M / 256 x H / 256, cols / 64 blocks
// each), so whole tiles leave SMs idle: 300 x 2040 are 16 tiles for 74 pairs.  The slices' sums are joined by a kernel of
// its own; its traffic, in units of a block's time (a third of a microsecond), is weighed against the shorter critical path.
// dW's many short tiles fill the gaps where there is a dW.  With few rows those are bound by their epilogue, which PAIR_STORE_LONG
// slows down, so no slice is then longer than an accumulator may sum.
int dx_split(int M, int H, int cols, bool with_dw) {
  const int tiles = ceil_div(M, kPairRows) * ceil_div(H, kPairMaxBN), blocks = ceil_div(cols, 64);
  const double even = (with_dw ? 2.0 : 1.0) * tiles * blocks / kPairsModel;          // dW is as much work as dX
  const long long slice_bytes = (long long)M * (long long)round_up((size_t)H, 32) * 4;
  const int fewest = with_dw && M <= kPairRows ? ceil_div(blocks, kPairStoreChunk) : 1, first = fewest * slice_bytes <= (512ll << 20) ? fewest : 1;
  double best = 0.0;
  int split = 1;
  for (int s = first; s == first || (s <= 16 && s * slice_bytes <= (512ll << 20) && blocks / s >= 16); ++s) {
    const double longest = (double)ceil_div(tiles * s, kPairsModel) * (ceil_div(blocks, s) + 8);
    const double cost = std::max(longest, even) + (s > 1 ? 10.0 + 2.0 * s * slice_bytes / 1.7e6 : 0.0);
    if (s == first || cost < 0.97 * best) { best = cost; split = s; }
  }
  return split;
}

// Operands whose rows miss TMA's 16 bytes.
struct Copies { bool x, w; };

Layout xent_layout(int M, int V, int H, Copies copies, bool backward) {
  Layout l{};
  size_t at = 0;
  const auto take = [&](size_t bytes) { const size_t p = at; at += round_up(bytes, 256); return p; };
  l.hp = (int)round_up((size_t)H, 64);     // whole blocks: every box is a wide one
  if (copies.x) l.x_copy = take((size_t)M * l.hp * 2);
  if (copies.w) l.w_copy = take((size_t)V * l.hp * 2);
  if (!backward) {
    const size_t tiles_n = ((size_t)V + kPairMaxBN - 1) / kPairMaxBN;
    l.partial = take(2 * tiles_n * M * sizeof(float2));
    l.target_logit = take((size_t)M * sizeof(float));
  } else {
    l.piece = xent_piece(M, V);
    l.pieces = (V + l.piece - 1) / l.piece;
    l.ld_dl = l.piece;
    l.ld_acc = (long long)round_up((size_t)H, 32);
    l.scale = take(2 * sizeof(float));
    l.dl = take((size_t)M * l.piece * 2);
    const int first = std::min(V, l.piece);
    l.max_split = std::max(dx_split(M, H, first, false), dx_split(M, H, first, true));
    l.acc_slice = (long long)M * l.ld_acc;
    if (l.pieces > 1 || l.max_split > 1) l.acc = take((size_t)l.max_split * l.acc_slice * sizeof(float));
  }
  l.total = at;
  return l;
}

bool misses_16_bytes(const void* p, long long ld) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0 || ld % 8 != 0; }
Copies needs_copies(const void* X, long long ldx, const void* W, long long ldw) { return {misses_16_bytes(X, ldx), misses_16_bytes(W, ldw)}; }

// Puts the copies in place of the operands.  A copy's lines end in zeros, so that they are whole blocks.
int make_copies(const Layout& l, Copies copies, uint8_t* ws, int M, int V, int H, const void** X, long long* ldx, int* inner_x, const void** W,
                long long* ldw, int* inner_w, cudaStream_t stream) {
  *inner_x = *inner_w = H;
  if (copies.x) {
    if (int rc = host_pad_rows16(*X, *ldx, ws + l.x_copy, M, H, l.hp, stream)) return rc;
    *X = ws + l.x_copy; *ldx = *inner_x = l.hp;
  }
  if (copies.w) {
    if (int rc = host_pad_rows16(*W, *ldw, ws + l.w_copy, V, H, l.hp, stream)) return rc;
    *W = ws + l.w_copy; *ldw = *inner_w = l.hp;
  }
  return MP_OK;
}

int check_args(const char* op, int dtype, int M, int V, int H, const void* X, long long ldx, const void* W, long long ldw,
               const void* target, int target_bytes) {
  if (dtype != MP_FP16 && dtype != MP_BF16) return host_fail(MP_ERR_INVALID_ARG, "%s: dtype must be MP_FP16 or MP_BF16", op);
  if (M < 0 || V <= 0 || H <= 0) return host_fail(MP_ERR_INVALID_ARG, "%s: needs M >= 0, V > 0, H > 0 (got %d, %d, %d)", op, M, V, H);
  if (V > (1 << 30) || M > (1 << 30) || H > (1 << 30)) return host_fail(MP_ERR_INVALID_ARG, "%s: extents above 2^30", op);
  if (ldx < H || ldw < H) return host_fail(MP_ERR_INVALID_ARG, "%s: row strides %lld and %lld below H = %d", op, ldx, ldw, H);
  if (target_bytes != 4 && target_bytes != 8) return host_fail(MP_ERR_INVALID_ARG, "%s: targets are int32 or int64", op);
  if (W == nullptr || (M > 0 && (X == nullptr || target == nullptr))) return host_fail(MP_ERR_INVALID_ARG, "%s: null pointer", op);
  return MP_OK;
}

int check_workspace(const char* op, void* ws, size_t have, size_t need) {
  if (need == 0) return MP_OK;
  if (ws == nullptr || have < need) return host_fail(MP_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", op, ws ? have : (size_t)0, need);
  if (reinterpret_cast<uintptr_t>(ws) & 255) return host_fail(MP_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", op);
  return MP_OK;
}

void shape_problem(PairProblem* q, int rows, int cols, int contraction, int bn, int a_mn, int b_mn, int group_m, int tile0) {
  q->rows = rows; q->cols = cols;
  q->kblocks = ceil_div(contraction, 64);
  q->bn = bn;
  q->tiles_m = ceil_div(rows, kPairRows);
  q->tiles_n = ceil_div(cols, bn);
  q->a_mn = a_mn; q->b_mn = b_mn;
  q->a_rows = a_mn ? 128 : std::min(128, (int)round_up((size_t)rows, 8));
  q->group_m = std::max(1, std::min(group_m, q->tiles_m));
  q->tile0 = tile0;
  q->split = 1;
  q->kb_per_split = q->kblocks;
}

template <int EPI>
int launch_pair(const HostDevice& d, PairParams& p, const PairMaps& maps, cudaStream_t stream) {
  auto kern = pair_gemm_kernel<EPI>;
  static bool ready[64] = {};
  if (!ready[d.index & 63]) {
    MP_HOST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem));
    ready[d.index & 63] = true;
  }
  const int bn = p.num_problems == 2 ? std::max(p.prob[0].bn, p.prob[1].bn) : p.prob[0].bn;
  p.kc = kStageBlocks;
  const int a_rows = p.num_problems == 2 ? 128 : p.prob[0].a_rows;
  p.stage_bytes = p.kc * (a_rows * 128 + bn / 2 * 128);
  p.stages = std::min(kPairMaxStages, (kPairSmem - 1024 - kPairBarBytes - (EPI == PAIR_LSE ? 0 : kPairStoreBytes)) / p.stage_bytes);
  p.status = d.status;
  const int pairs = std::max(1, std::min(p.total_tiles, d.sms / 2));
  return host_launch(kern, 2 * pairs, kPairThreads, kPairSmem, stream, maps, p);
}

// Row tiles that run side by side against one column tile: their operand rows should stay in L2 while the columns pass.
int group_rows(long long row_bytes) {
  const long long tile = row_bytes * kPairRows;
  return (int)std::max<long long>(1, std::min<long long>(64, (48ll << 20) / std::max<long long>(tile, 1)));
}

}  // namespace

extern "C" {

int mp_linear_xent_workspace(int dtype, int M, int V, int H, const void* X, long long ldx, const void* W, long long ldw,
                             int backward, size_t* bytes) {
  if (bytes == nullptr) return host_fail(MP_ERR_INVALID_ARG, "mp_linear_xent_workspace: null pointer");
  if (int rc = check_args("mp_linear_xent_workspace", dtype, M, V, H, X ? X : W, ldx, W, ldw, W, 8)) return rc;
  *bytes = M == 0 ? 0 : xent_layout(M, V, H, needs_copies(X, ldx, W, ldw), backward != 0).total;
  return MP_OK;
}

int mp_linear_xent(int dtype, int M, int V, int H, const void* X, long long ldx, const void* W, long long ldw, const void* target,
                   int target_bytes, long long ignore_index, float* loss, float* lse, void* workspace, size_t workspace_bytes,
                   void* stream_) {
  const char* op = "mp_linear_xent";
  if (int rc = check_args(op, dtype, M, V, H, X, ldx, W, ldw, target, target_bytes)) return rc;
  if (M == 0) return MP_OK;
  if (loss == nullptr || lse == nullptr) return host_fail(MP_ERR_INVALID_ARG, "%s: null output", op);
  const Copies copies = needs_copies(X, ldx, W, ldw);
  const Layout l = xent_layout(M, V, H, copies, false);
  if (int rc = check_workspace(op, workspace, workspace_bytes, l.total)) return rc;
  HostDevice d;
  if (int rc = host_device(&d)) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  int inner_x, inner_w;
  if (int rc = make_copies(l, copies, ws, M, V, H, &X, &ldx, &inner_x, &W, &ldw, &inner_w, stream)) return rc;
  PairParams p{};
  p.num_problems = 1;
  shape_problem(&p.prob[0], M, V, H, kPairMaxBN, 0, 0, group_rows((long long)H * 2), 0);
  p.total_tiles = p.prob[0].tiles_m * p.prob[0].tiles_n;
  p.bf16 = dtype == MP_BF16;
  p.target = target; p.target64 = target_bytes == 8; p.ignore_index = ignore_index;
  p.partial = reinterpret_cast<float2*>(ws + l.partial);
  p.target_logit = reinterpret_cast<float*>(ws + l.target_logit);
  PairMaps maps{};
  if (int rc = operand_maps(&maps.a[0], X, inner_x, M, ldx, p.prob[0].a_rows, kStageBlocks, &p.prob[0].a_wide)) return rc;
  if (int rc = operand_maps(&maps.b[0], W, inner_w, V, ldw, p.prob[0].bn / 2, kStageBlocks, &p.prob[0].b_wide)) return rc;
  if (int rc = launch_pair<PAIR_LSE>(d, p, maps, stream)) return rc;
  return host_launch(xent_join_kernel, ceil_div(M, 32), 1024, 0, stream, p.partial, 2 * p.prob[0].tiles_n, M, p.target_logit, target, p.target64,
                ignore_index, V, loss, lse);
}

int mp_linear_xent_grad(int dtype, int M, int V, int H, const void* X, long long ldx, const void* W, long long ldw, const void* target,
                        int target_bytes, long long ignore_index, const float* lse, const float* grad_loss, void* dX, void* dW,
                        void* workspace, size_t workspace_bytes, void* stream_) {
  const char* op = "mp_linear_xent_grad";
  if (int rc = check_args(op, dtype, M, V, H, X, ldx, W, ldw, target, target_bytes)) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (dX == nullptr && dW == nullptr) return MP_OK;
  HostDevice d;
  if (M == 0) {                                       // a sum over no tokens
    if (dW == nullptr) return MP_OK;
    if (int rc = host_device(&d)) return rc;
    MP_HOST_CUDA_TRY(cudaMemsetAsync(dW, 0, (size_t)V * H * 2, stream));
    return MP_OK;
  }
  if (lse == nullptr || grad_loss == nullptr) return host_fail(MP_ERR_INVALID_ARG, "%s: null pointer", op);
  const Copies copies = needs_copies(X, ldx, W, ldw);
  const Layout l = xent_layout(M, V, H, copies, true);
  if (int rc = check_workspace(op, workspace, workspace_bytes, l.total)) return rc;
  if (int rc = host_device(&d)) return rc;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  int inner_x, inner_w;
  if (int rc = make_copies(l, copies, ws, M, V, H, &X, &ldx, &inner_x, &W, &ldw, &inner_w, stream)) return rc;
  float* scale = reinterpret_cast<float*>(ws + l.scale);
  unsigned* counter = reinterpret_cast<unsigned*>(ws + l.scale) + 1;
  uint16_t* dl = reinterpret_cast<uint16_t*>(ws + l.dl);
  // slices of the same length in every piece: a short last piece leaves the last ones without work, and none is added to
  // that the first piece has not written
  const int split = dX == nullptr ? 1 : dx_split(M, H, std::min(V, l.piece), dW != nullptr);
  const int kb_per_split = (int)round_up((size_t)ceil_div(ceil_div(std::min(V, l.piece), 64), split), kStageBlocks);
  const int bf16 = dtype == MP_BF16, target64 = target_bytes == 8;

  int slices = 0;                                     // of dX, waiting to be joined
  for (int i = 0; i < l.pieces; ++i) {
    const int col0 = i * l.piece, cols = std::min(l.piece, V - col0);
    const uint16_t* Wp = reinterpret_cast<const uint16_t*>(W) + (long long)col0 * ldw;
    PairMaps maps{};
    {
      PairParams p{};
      p.num_problems = 1;
      shape_problem(&p.prob[0], M, cols, H, kPairMaxBN, 0, 0, group_rows((long long)H * 2), 0);
      p.total_tiles = p.prob[0].tiles_m * p.prob[0].tiles_n;
      p.bf16 = bf16;
      p.target = target; p.target64 = target64; p.ignore_index = ignore_index;
      p.col0 = col0; p.lse = lse; p.grad_loss = grad_loss; p.vocab = V; p.scale_out = scale; p.next_unit = counter; p.dlogits = dl; p.ld_dl = l.ld_dl;
      if (int rc = operand_maps(&maps.a[0], X, inner_x, M, ldx, p.prob[0].a_rows, kStageBlocks, &p.prob[0].a_wide)) return rc;
      if (int rc = operand_maps(&maps.b[0], Wp, inner_w, cols, ldw, p.prob[0].bn / 2, kStageBlocks, &p.prob[0].b_wide)) return rc;
      if (int rc = launch_pair<PAIR_DLOGITS>(d, p, maps, stream)) return rc;
    }
    PairParams p{};
    p.bf16 = bf16;
    p.next_unit = counter;
    p.scale = scale;
    int n = 0;
    if (dX != nullptr) {                              // dX[M, H] (+)= d[M, cols] W[cols, H]
      PairProblem& q = p.prob[n];
      shape_problem(&q, M, H, cols, kPairMaxBN, 0, 1, 8, p.total_tiles);
      q.acc32 = reinterpret_cast<float*>(ws + l.acc);
      q.ld_acc = l.ld_acc;
      q.acc_slice = l.acc_slice;
      q.add_acc32 = i > 0;
      if (split > 1) {
        q.kb_per_split = kb_per_split;
        q.split = ceil_div(q.kblocks, kb_per_split);
        if (i == 0) slices = q.split;
      } else if (i == l.pieces - 1) {
        q.out16 = dX; q.ld_out = H;
      }
      if (int rc = operand_maps(&maps.a[n], dl, cols, M, l.ld_dl, q.a_rows, kStageBlocks, &q.a_wide)) return rc;
      if (int rc = operand_maps(&maps.b[n], Wp, inner_w, cols, ldw, kStageBlocks * 64, q.bn / 2 / 64, &q.b_wide)) return rc;
      p.total_tiles += q.tiles_m * q.tiles_n * q.split;
      ++n;
    }
    if (dW != nullptr) {                              // dW[cols, H] = d^T[cols, M] X[M, H]
      PairProblem& q = p.prob[n];
      shape_problem(&q, cols, H, M, kPairMaxBN, 1, 1, 8, p.total_tiles);
      q.out16 = reinterpret_cast<uint16_t*>(dW) + (long long)col0 * H;
      q.ld_out = H;
      if (int rc = operand_maps(&maps.a[n], dl, cols, M, l.ld_dl, kStageBlocks * 64, 128 / 64, &q.a_wide)) return rc;
      if (int rc = operand_maps(&maps.b[n], X, inner_x, M, ldx, kStageBlocks * 64, q.bn / 2 / 64, &q.b_wide)) return rc;
      p.total_tiles += q.tiles_m * q.tiles_n;
      ++n;
    }
    p.num_problems = n;
    bool chunks = false;
    for (int j = 0; j < n; ++j) chunks |= p.prob[j].kb_per_split > kPairStoreChunk;
    if (int rc = chunks ? launch_pair<PAIR_STORE_LONG>(d, p, maps, stream) : launch_pair<PAIR_STORE>(d, p, maps, stream)) return rc;
  }
  if (slices > 0) {
    const long long threads = (long long)M * (l.ld_acc / 4);
    return host_launch(xent_dx_kernel, (int)((threads + 255) / 256), 256, 0, stream, reinterpret_cast<const float*>(ws + l.acc), slices, l.acc_slice,
                  l.ld_acc, M, H, scale, reinterpret_cast<uint16_t*>(dX), bf16);
  }
  return MP_OK;
}

}  // extern "C"
