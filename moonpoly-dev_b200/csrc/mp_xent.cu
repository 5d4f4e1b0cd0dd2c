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
// loss and logsumexp of every row from the partial (max, sum) pairs; 32 rows x 32 groups of partials per block.
__global__ void __launch_bounds__(1024) xent_join_kernel(const float2* partial, int num, int rows, const float* target_logit,
                                                         const void* target, int target64, long long ignore_index, int vocab,
                                                         float* loss, float* lse) {
  __shared__ float sm[32][33], ss[32][33];
  const int rx = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + rx;
  float m = -INFINITY, s = 0.0f;
  if (row < rows) {
    for (int i = g; i < num; i += 32) {
      const float2 v = partial[(size_t)i * rows + row];
      const float mn = fmaxf(m, v.x);
      if (mn != -INFINITY) {                       // two empty pieces would give exp(-inf + inf)
        s = s * exp2_approx((m - mn) * kLog2e) + v.y * exp2_approx((v.x - mn) * kLog2e);
        m = mn;
      } else {
        s += v.y;                                  // 0, or NaN from a row of NaN
      }
    }
  }
  sm[g][rx] = m;
  ss[g][rx] = s;
  __syncthreads();
  if (g != 0 || row >= rows) return;
  float top = -INFINITY;
  for (int i = 0; i < 32; ++i) top = fmaxf(top, sm[i][rx]);
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  for (int i = 0; i < 32; ++i) sum += ss[i][rx] * exp2_approx((sm[i][rx] - base) * kLog2e);
  const float logsum = logf(sum);
  lse[row] = base + logsum;
  const long long t = target64 ? reinterpret_cast<const long long*>(target)[row] : reinterpret_cast<const int*>(target)[row];
  if (t == ignore_index) loss[row] = 0.0f;
  else if (t < 0 || t >= vocab) loss[row] = NAN;   // no such entry: loud, and nothing is read out of range
  else loss[row] = logsum + (base - target_logit[row]);   // small losses keep their digits: no large lse is formed
}

// Row factors of d and the scale of the products.  d is parked in 16 bits, so the largest |g| is divided out (a mean over
// the tokens then rounds exactly: the factors are 1) and, for fp16, replaced by 2^15: a probability of 2e-9 is still a
// normal fp16 number beside a one.  One block: the rows of a training batch are a few kilobytes.
__global__ void __launch_bounds__(1024) xent_coef_kernel(const float* grad_loss, const void* target, int target64,
                                                         long long ignore_index, int vocab, int rows, int bf16, float* coef, float* scale) {
  __shared__ float red[32];
  float g = 0.0f;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const long long t = target64 ? reinterpret_cast<const long long*>(target)[i] : reinterpret_cast<const int*>(target)[i];
    if (t != ignore_index) {
      const float a = fabsf(grad_loss[i]);
      if (a < INFINITY) g = fmaxf(g, a);           // infinities and NaN go through as they are
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = g;
  __syncthreads();
  g = red[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
  if (g == 0.0f) g = 1.0f;
  const float up = bf16 ? 1.0f : 32768.0f;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const long long t = target64 ? reinterpret_cast<const long long*>(target)[i] : reinterpret_cast<const int*>(target)[i];
    const bool bad = t < 0 || t >= vocab;
    coef[i] = t == ignore_index ? 0.0f : bad ? NAN : grad_loss[i] / g * up;
  }
  if (threadIdx.x == 0) *scale = g / up;
}

// ------------------------------------------------------------------------------------------------------------ problem
struct Xent {
  int dtype, M, V, H;
  const void* X; long long ldx;
  const void* W; long long ldw;
  const void* target; int target64;
  long long ignore_index;
};

// Sizes that follow from the shape alone, so that the workspace query and the call agree.
struct Layout {
  size_t x_copy, w_copy;                  // aligned copies of operands whose rows miss TMA's 16 bytes
  size_t partial, target_logit;           // forward
  size_t coef, dl, acc;                   // gradients
  int hp, piece, pieces;
  long long ld_acc, ld_dl;
  size_t total;
};

// Vocabulary entries per piece of the gradient.
int xent_piece(int M, int V) {
  const long long rows = std::max<long long>(round_up((size_t)M, 256), 256);
  long long piece = (256ll << 20) / (2 * rows) / 256 * 256;
  piece = std::max<long long>(piece, 4096);
  return (int)std::min<long long>(piece, (long long)round_up((size_t)V, 256));
}

Layout xent_layout(int M, int V, int H, bool copies, bool backward) {
  Layout l{};
  size_t at = 0;
  const auto take = [&](size_t bytes) { const size_t p = at; at += round_up(bytes, 256); return p; };
  l.hp = (int)round_up((size_t)H, 8);
  if (copies) {
    l.x_copy = take((size_t)M * l.hp * 2);
    l.w_copy = take((size_t)V * l.hp * 2);
  }
  if (!backward) {
    const size_t tiles_n = ((size_t)V + kPairMaxBN - 1) / kPairMaxBN;
    l.partial = take(2 * tiles_n * M * sizeof(float2));
    l.target_logit = take((size_t)M * sizeof(float));
  } else {
    l.piece = xent_piece(M, V);
    l.pieces = (V + l.piece - 1) / l.piece;
    l.ld_dl = l.piece;
    l.ld_acc = (long long)round_up((size_t)H, 32);
    l.coef = take(((size_t)M + 64) * sizeof(float));
    l.dl = take((size_t)M * l.piece * 2);
    if (l.pieces > 1) l.acc = take((size_t)M * l.ld_acc * sizeof(float));
  }
  l.total = at;
  return l;
}

bool needs_copies(const void* X, long long ldx, const void* W, long long ldw) {
  return ((reinterpret_cast<uintptr_t>(X) | reinterpret_cast<uintptr_t>(W)) & 15) != 0 || ldx % 8 != 0 || ldw % 8 != 0;
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

// 64-element contraction blocks per pipeline stage.
constexpr int kStageBlocks = 2;

// TMA view of a row-major 16-bit matrix as a K-major operand of which a CTA takes `rows_cta` rows, or as an MN-major one of
// which it takes `rows_cta` columns.
int operand_map(CUtensorMap* tm, const void* ptr, long long inner, long long rows, long long ld, bool mn, int rows_cta, int* wide) {
  const int kc = kStageBlocks;
  *wide = inner % 64 == 0 && kc > 1;
  if (*wide) return host_tmap_blocks(tm, ptr, inner, rows, ld * 2, mn ? kc * 64 : rows_cta, mn ? rows_cta / 64 : kc);
  return host_tmap(tm, kTmap16, ptr, inner, rows, ld * 2, 64, mn ? kc * 64 : rows_cta, 128);
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

void shape_problem(PairProblem* q, int rows, int cols, int contraction, int bn, int a_mn, int b_mn, int group_m, int tile0) {
  q->rows = rows; q->cols = cols;
  q->kblocks = ceil_div(contraction, 64);
  q->bn = bn;
  q->tiles_m = ceil_div(rows, kPairRows);
  q->tiles_n = ceil_div(cols, bn);
  q->a_mn = a_mn; q->b_mn = b_mn;
  q->group_m = std::max(1, std::min(group_m, q->tiles_m));
  q->tile0 = tile0;
}

template <int EPI>
int launch_pair(const HostDevice& d, PairParams& p, const CUtensorMap (&tm)[4], cudaStream_t stream) {
  auto kern = pair_gemm_kernel<EPI>;
  static bool ready[64] = {};
  if (!ready[d.index & 63]) {
    MP_HOST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem));
    ready[d.index & 63] = true;
  }
  const int bn = p.num_problems == 2 ? std::max(p.prob[0].bn, p.prob[1].bn) : p.prob[0].bn;
  p.kc = kStageBlocks;
  p.stage_bytes = p.kc * (kPairABytes + bn / 2 * 128);
  p.stages = std::min(kPairMaxStages, (kPairSmem - 1024 - 256) / p.stage_bytes);
  p.status = d.status;
  const int pairs = std::max(1, std::min(p.total_tiles, d.sms / 2));
  kern<<<2 * pairs, kPairThreads, kPairSmem, stream>>>(tm[0], tm[1], tm[2], tm[3], p);
  MP_HOST_CUDA_TRY(cudaGetLastError());
  host_count_launches(1);
  return MP_OK;
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
  const bool copies = needs_copies(X, ldx, W, ldw);
  const Layout l = xent_layout(M, V, H, copies, false);
  if (int rc = check_workspace(op, workspace, workspace_bytes, l.total)) return rc;
  HostDevice d;
  if (int rc = host_device(&d)) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  if (copies) {
    if (int rc = host_pad_rows16(X, ldx, ws + l.x_copy, M, H, l.hp, stream)) return rc;
    if (int rc = host_pad_rows16(W, ldw, ws + l.w_copy, V, H, l.hp, stream)) return rc;
    X = ws + l.x_copy; W = ws + l.w_copy; ldx = ldw = l.hp;
  }
  PairParams p{};
  p.num_problems = 1;
  shape_problem(&p.prob[0], M, V, H, kPairMaxBN, 0, 0, group_rows((long long)H * 2), 0);
  p.total_tiles = p.prob[0].tiles_m * p.prob[0].tiles_n;
  p.bf16 = dtype == MP_BF16;
  p.target = target; p.target64 = target_bytes == 8; p.ignore_index = ignore_index;
  p.partial = reinterpret_cast<float2*>(ws + l.partial);
  p.target_logit = reinterpret_cast<float*>(ws + l.target_logit);
  CUtensorMap tm[4];
  if (int rc = operand_map(&tm[0], X, H, M, ldx, false, 128, &p.prob[0].a_wide)) return rc;
  if (int rc = operand_map(&tm[1], W, H, V, ldw, false, p.prob[0].bn / 2, &p.prob[0].b_wide)) return rc;
  tm[2] = tm[0]; tm[3] = tm[1];
  if (int rc = launch_pair<PAIR_LSE>(d, p, tm, stream)) return rc;
  xent_join_kernel<<<ceil_div(M, 32), 1024, 0, stream>>>(p.partial, 2 * p.prob[0].tiles_n, M, p.target_logit, target, p.target64,
                                                         ignore_index, V, loss, lse);
  MP_HOST_CUDA_TRY(cudaGetLastError());
  host_count_launches(1);
  return MP_OK;
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
  const bool copies = needs_copies(X, ldx, W, ldw);
  const Layout l = xent_layout(M, V, H, copies, true);
  if (int rc = check_workspace(op, workspace, workspace_bytes, l.total)) return rc;
  if (int rc = host_device(&d)) return rc;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  if (copies) {
    if (int rc = host_pad_rows16(X, ldx, ws + l.x_copy, M, H, l.hp, stream)) return rc;
    if (int rc = host_pad_rows16(W, ldw, ws + l.w_copy, V, H, l.hp, stream)) return rc;
    X = ws + l.x_copy; W = ws + l.w_copy; ldx = ldw = l.hp;
  }
  float* coef = reinterpret_cast<float*>(ws + l.coef);
  float* scale = coef + M;
  uint16_t* dl = reinterpret_cast<uint16_t*>(ws + l.dl);
  const int bf16 = dtype == MP_BF16, target64 = target_bytes == 8;
  xent_coef_kernel<<<1, 1024, 0, stream>>>(grad_loss, target, target64, ignore_index, V, M, bf16, coef, scale);
  MP_HOST_CUDA_TRY(cudaGetLastError());
  host_count_launches(1);

  for (int i = 0; i < l.pieces; ++i) {
    const int col0 = i * l.piece, cols = std::min(l.piece, V - col0);
    const uint16_t* Wp = reinterpret_cast<const uint16_t*>(W) + (long long)col0 * ldw;
    CUtensorMap tm[4];
    {
      PairParams p{};
      p.num_problems = 1;
      shape_problem(&p.prob[0], M, cols, H, kPairMaxBN, 0, 0, group_rows((long long)H * 2), 0);
      p.total_tiles = p.prob[0].tiles_m * p.prob[0].tiles_n;
      p.bf16 = bf16;
      p.target = target; p.target64 = target64; p.ignore_index = ignore_index;
      p.col0 = col0; p.lse = lse; p.coef = coef; p.dlogits = dl; p.ld_dl = l.ld_dl;
      if (int rc = operand_map(&tm[0], X, H, M, ldx, false, 128, &p.prob[0].a_wide)) return rc;
      if (int rc = operand_map(&tm[1], Wp, H, cols, ldw, false, p.prob[0].bn / 2, &p.prob[0].b_wide)) return rc;
      tm[2] = tm[0]; tm[3] = tm[1];
      if (int rc = launch_pair<PAIR_DLOGITS>(d, p, tm, stream)) return rc;
    }
    PairParams p{};
    p.bf16 = bf16;
    int n = 0;
    if (dX != nullptr) {                              // dX[M, H] (+)= d[M, cols] W[cols, H]
      PairProblem& q = p.prob[n];
      shape_problem(&q, M, H, cols, kPairMaxBN, 0, 1, 8, p.total_tiles);
      q.acc32 = reinterpret_cast<float*>(ws + l.acc);
      q.ld_acc = l.ld_acc;
      q.add_acc32 = i > 0;
      if (i == l.pieces - 1) { q.out16 = dX; q.ld_out = H; q.scale = scale; }
      if (int rc = operand_map(&tm[2 * n], dl, cols, M, l.ld_dl, false, 128, &q.a_wide)) return rc;
      if (int rc = operand_map(&tm[2 * n + 1], Wp, H, cols, ldw, true, q.bn / 2, &q.b_wide)) return rc;
      p.total_tiles += q.tiles_m * q.tiles_n;
      ++n;
    }
    if (dW != nullptr) {                              // dW[cols, H] = d^T[cols, M] X[M, H]
      PairProblem& q = p.prob[n];
      shape_problem(&q, cols, H, M, kPairMaxBN, 1, 1, 8, p.total_tiles);
      q.out16 = reinterpret_cast<uint16_t*>(dW) + (long long)col0 * H;
      q.ld_out = H;
      q.scale = scale;
      if (int rc = operand_map(&tm[2 * n], dl, cols, M, l.ld_dl, true, 128, &q.a_wide)) return rc;
      if (int rc = operand_map(&tm[2 * n + 1], X, H, M, ldx, true, q.bn / 2, &q.b_wide)) return rc;
      p.total_tiles += q.tiles_m * q.tiles_n;
      ++n;
    }
    p.num_problems = n;
    if (n == 1) { tm[2] = tm[0]; tm[3] = tm[1]; }
    if (int rc = launch_pair<PAIR_STORE>(d, p, tm, stream)) return rc;
  }
  return MP_OK;
}

}  // extern "C"
