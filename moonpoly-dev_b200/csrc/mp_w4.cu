// Linear with 4-bit weights (mp_w4_pack, mp_linear_w4, mp_linear_w4_grad_input): argument checks, choice of the kernel,
// workspaces, launches.  The kernels and the packed format are in mp_w4.cuh.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/moonpoly_abi.h"
#include "mp_host.h"
#include "mp_w4.cuh"

namespace {

using namespace mp;

size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
int ceil_div(int a, int b) { return (a + b - 1) / b; }

constexpr int kW4StreamMaxTokens = 16;
constexpr int kSmsModel = 148;            // workspace sizes must not depend on the device that is asked

struct Plan {
  bool stream, with_table;
  int bn, tiles_m, tiles_n, steps, split, steps_per_split;
  int stages, stage_bytes, raw_slots;
  size_t copy, partial, table, total;     // workspace: aligned copy of the tokens, partial sums, group words
  long long ld_copy, ld_partial;
};

bool tokens_aligned(const void* x, long long ld) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld % 8 == 0; }

// Slots of the ring of packed weights: what three stages leave of the shared memory, but never three.  The two unpacking groups
// take turns, and a wait tells a slot's fill from the one before it by the parity of the phase alone, so a group may wait for a
// fill only where the one before it is known to have landed.  With an even number of slots that one was the group's own.  With
// five, it was turn T - 5 of the other group: the group's last stage of turn T - 2 was free only after the product of the step
// three before it, turns T - 4 ... T - 2 hold at least three steps, so turn T - 5 has been multiplied.  Three slots go wrong
// where a turn of one step (the end of a unit with an odd number of steps) comes into it.
int w4_raw_slots(int stages, int stage_bytes) {
  const int room = std::min(kW4MaxRawSlots, (kPairSmem - 1024 - 256 - stages * stage_bytes) / kW4RawBytes);
  return room == 3 ? 2 : room;
}

// rows = output features of this direction, contraction = input features.
Plan w4_plan(int T, int N, int K, int group_size, bool grad, bool copy_tokens) {
  Plan p{};
  const int rows = grad ? K : N, contraction = grad ? N : K;
  p.stream = !grad && T <= kW4StreamMaxTokens;
  if (copy_tokens) {
    p.ld_copy = (long long)round_up((size_t)contraction, 64);      // whole blocks: every box is a wide one
    p.copy = p.total;
    p.total += round_up((size_t)T * p.ld_copy * 2, 256);
  }
  if (p.stream) return p;
  p.steps = ceil_div(contraction, 128);
  const int slots = kSmsModel / 2;
  p.tiles_m = ceil_div(rows, kPairRows);
  // Tokens per tile (a multiple of 32) and slices of the contraction: the choice whose longest pair is done first.  A step
  // of a tile costs four cycles per token on the tensor cores, or the 900 of the unpacking; a slice at least four steps, and
  // eight for its sums to be written and joined.
  double best = 0.0;
  const int whole = std::min(256, (int)round_up((size_t)T, 32));
  for (int bn = whole; bn >= std::min(160, whole); bn -= 32) {
    const int tiles = p.tiles_m * ceil_div(T, bn);
    for (int split = 1; split <= 16 && (split == 1 || p.steps / split >= 4) && (split == 1 || tiles * split <= slots); ++split) {
      const int each = ceil_div(p.steps, split);
      const double cost = (double)ceil_div(tiles * ceil_div(p.steps, each), slots) * (each + (split > 1 ? 8 : 0)) * std::max(4 * bn + 100, 900);
      if (best == 0.0 || cost < best) { best = cost; p.bn = bn; p.split = split; }
    }
  }
  p.tiles_n = ceil_div(T, p.bn);
  p.steps_per_split = ceil_div(p.steps, p.split);
  p.split = ceil_div(p.steps, p.steps_per_split);
  // three stages, and the rest of the shared memory for packed bytes on their way from HBM
  p.stages = 3;
  p.stage_bytes = kW4ABytes + p.bn / 2 * 256;
  p.raw_slots = w4_raw_slots(p.stages, p.stage_bytes);
  // The transposed group words cost a kernel of 3 us.  They pay where the weight is unpacked for several token tiles, and with
  // fine groups always (28672 x 4096, groups of 64, 17 tokens: 45 us against 58).
  p.with_table = p.tiles_n > 1 || group_size < 128;
  if (p.with_table) {
    p.table = p.total;
    p.total += round_up((size_t)ceil_div(K, group_size) * N * 4, 256);
  }
  if (p.split > 1) {
    p.ld_partial = (long long)round_up((size_t)rows, 32);
    p.partial = p.total;
    p.total += round_up((size_t)p.split * T * p.ld_partial * 4, 256);
  }
  return p;
}

constexpr int kMaxExtent = 1 << 28;

int check_shape(const char* op, int M, int N, int K, int group_size) {
  if (M < 0 || N <= 0 || K <= 0 || M > kMaxExtent || N > kMaxExtent || K > kMaxExtent)
    return host_fail(MP_ERR_INVALID_ARG, "%s: needs M >= 0, N > 0, K > 0, none above 2^28 (got %d, %d, %d)", op, M, N, K);
  if (K % 32 != 0) return host_fail(MP_ERR_UNALIGNED_K, "%s: K = %d is not a multiple of 32", op, K);
  if (group_size < 32 || (group_size & (group_size - 1)) != 0)
    return host_fail(MP_ERR_INVALID_ARG, "%s: group_size %d is not a power of two of at least 32", op, group_size);
  return MP_OK;
}

int check_args(const char* op, int dtype, int M, int N, int K, const void* x, long long ldx, int width, const uint32_t* packed,
               const void* scales, int group_size) {
  if (dtype != MP_FP16 && dtype != MP_BF16) return host_fail(MP_ERR_INVALID_ARG, "%s: dtype must be MP_FP16 or MP_BF16", op);
  if (int rc = check_shape(op, M, N, K, group_size)) return rc;
  if (ldx < width) return host_fail(MP_ERR_INVALID_ARG, "%s: row stride %lld below the row's %d elements", op, ldx, width);
  if (packed == nullptr || scales == nullptr || (M > 0 && x == nullptr)) return host_fail(MP_ERR_INVALID_ARG, "%s: null pointer", op);
  if (reinterpret_cast<uintptr_t>(packed) & 15) return host_fail(MP_ERR_INVALID_ARG, "%s: the packed weight must be 16-byte aligned", op);
  return MP_OK;
}

W4Weight weight_of(int N, int K, const uint32_t* packed, const void* scales, const uint8_t* zeros, int group_size) {
  W4Weight w{};
  w.packed = reinterpret_cast<const uint4*>(packed);
  w.scale = reinterpret_cast<const uint16_t*>(scales);
  w.zero = zeros;
  w.N = N; w.K = K;
  w.blocks = ceil_div(K, 128);
  w.groups = ceil_div(K, group_size);
  for (w.shift = 0; (32 << w.shift) < group_size; ++w.shift) {}
  return w;
}

template <bool BF16, int NT, int GPB>
int launch_stream(const HostDevice& d, const W4StreamParams& p, cudaStream_t stream) {
  const W4Weight& w = p.w;
  // One CTA per SM; more, in waves, where the parked sums of a share and its group words would leave no room for a ring of
  // four blocks.  Rows with so many groups that eight waves do not do it read them from global memory.
  constexpr size_t kBlock = (size_t)kW4StreamWarps * 1024;
  const int one = std::min(ceil_div(w.N, 16), d.sms);
  int ctas = one;
  size_t sums = 0, staged = 0;
  const auto shape = [&](int c) {
    const int rows = ceil_div(w.N, c), tiles = ceil_div(rows, 16);
    // shares are `rows` or `rows` - 1 long, and the shorter may be a single tile, whose sums are parked 16 times
    sums = (size_t)std::max(tiles * 8, 16) * NT * 512;
    staged = (size_t)tiles * 16 * w.groups * 4;
    ctas = c;
  };
  bool stage = false;
  for (int waves = 1; waves <= 8 && !stage; ++waves) {
    shape(one * waves);
    stage = 4 * kBlock + sums + staged <= (size_t)kPairSmem;
  }
  if (!stage)
    for (int waves = 1; shape(one * waves), 4 * kBlock + sums > (size_t)kPairSmem; ++waves) {}
  const size_t fixed = sums + (stage ? staged : 0);
  const bool deep = 8 * kBlock + fixed <= (size_t)kPairSmem;
  auto kern = stage ? (deep ? w4_stream_kernel<BF16, NT, GPB, 8, true> : w4_stream_kernel<BF16, NT, GPB, 4, true>)
                    : (deep ? w4_stream_kernel<BF16, NT, GPB, 8, false> : w4_stream_kernel<BF16, NT, GPB, 4, false>);
  static bool ready[64][4] = {};
  bool& done = ready[d.index & 63][stage * 2 + deep];
  if (!done) {
    MP_HOST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem));
    done = true;
  }
  return host_launch(kern, ctas, kW4StreamWarps * 32, (deep ? 8 : 4) * kBlock + fixed, stream, p);
}

template <bool BF16, int NT>
int run_stream_t(const HostDevice& d, const W4StreamParams& p, cudaStream_t stream) {
  return p.w.shift >= 2 ? launch_stream<BF16, NT, 1>(d, p, stream) : p.w.shift == 1 ? launch_stream<BF16, NT, 2>(d, p, stream)
                                                                                   : launch_stream<BF16, NT, 4>(d, p, stream);
}

template <bool BF16>
int run_stream(const HostDevice& d, const W4StreamParams& p, cudaStream_t stream) {
  return p.T <= 8 ? run_stream_t<BF16, 1>(d, p, stream) : run_stream_t<BF16, 2>(d, p, stream);
}

template <bool BF16>
int run_mma(const HostDevice& d, const Plan& l, const W4Weight& w, bool grad, int T, const void* x, long long ldx, int inner, const void* bias,
             void* out, uint8_t* ws, cudaStream_t stream) {
  W4PairParams p{};
  p.w = w;
  p.grad = grad;
  p.rows = grad ? w.K : w.N;
  p.T = T;
  p.steps = l.steps;
  p.tiles_m = l.tiles_m; p.tiles_n = l.tiles_n; p.bn = l.bn;
  p.split = l.split; p.steps_per_split = l.steps_per_split;
  p.out = reinterpret_cast<uint16_t*>(out);
  p.ldo = p.rows;
  p.bias = reinterpret_cast<const uint16_t*>(bias);
  p.partial = reinterpret_cast<float*>(ws + l.partial);
  p.ld_partial = l.ld_partial;
  p.status = d.status;
  p.stages = l.stages; p.stage_bytes = l.stage_bytes; p.raw_slots = l.raw_slots;
  OperandMaps tokens;
  CUtensorMap tmW;
  if (int rc = operand_maps(&tokens, x, inner, T, ldx, l.bn / 2, 2, &p.b_wide)) return rc;
  if (l.with_table) {
    p.table = reinterpret_cast<const uint32_t*>(ws + l.table);
    p.ld_table = w.N;
    const int across = ceil_div(w.N, 32);
    if (int rc = host_launch(w4_table_kernel, across * ceil_div(w.groups, 32), 256, 0, stream, w.scale, w.zero, w.N, w.groups, across,
                                  reinterpret_cast<uint32_t*>(ws + l.table), w.N)) return rc;
  }
  const int line = grad ? 64 : 128;                      // packed bytes per row and box
  if (int rc = host_tmap(&tmW, kTmapByte, w.packed, (long long)w.blocks * 64, w.N, (long long)w.blocks * 64, line, 128, line)) return rc;
  const bool fine = w.shift < 2;
  auto kern = fine ? w4_mma_kernel<BF16, true> : w4_mma_kernel<BF16, false>;
  static bool ready[64][2] = {};
  bool& done = ready[d.index & 63][fine];
  if (!done) {
    MP_HOST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem));
    done = true;
  }
  const int pairs = std::max(1, std::min(p.tiles_m * p.tiles_n * p.split, d.sms / 2));
  if (int rc = host_launch(kern, 2 * pairs, kW4Threads, kPairSmem, stream, tokens, tmW, p)) return rc;
  if (p.split > 1) {
    const long long threads = (long long)T * (l.ld_partial / 4);
    return host_launch(w4_reduce_kernel<BF16>, (int)((threads + 255) / 256), 256, 0, stream, p.partial, p.split, T, p.rows, p.ld_partial,
                            p.bias, p.out, p.ldo);
  }
  return MP_OK;
}

int run_w4(const char* op, bool grad, int dtype, int M, int N, int K, const void* X, long long ldx, const uint32_t* packed, const void* scales,
           const uint8_t* zeros, int group_size, const void* bias, void* out, void* workspace, size_t workspace_bytes, void* stream_) {
  const int width = grad ? N : K;
  int inner = width;
  if (int rc = check_args(op, dtype, M, N, K, X, ldx, width, packed, scales, group_size)) return rc;
  if (M == 0) return MP_OK;
  if (out == nullptr) return host_fail(MP_ERR_INVALID_ARG, "%s: null output", op);
  const bool copy = !tokens_aligned(X, ldx);
  const Plan l = w4_plan(M, N, K, group_size, grad, copy);
  if (l.total > 0) {
    if (workspace == nullptr || workspace_bytes < l.total)
      return host_fail(MP_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", op, workspace ? workspace_bytes : (size_t)0, l.total);
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return host_fail(MP_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", op);
  }
  HostDevice d;
  if (int rc = host_device(&d)) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  if (copy) {
    if (int rc = host_pad_rows16(X, ldx, ws + l.copy, M, width, (int)l.ld_copy, stream)) return rc;
    X = ws + l.copy;
    ldx = l.ld_copy;
    inner = (int)l.ld_copy;                              // its lines end in zeros
  }
  const W4Weight w = weight_of(N, K, packed, scales, zeros, group_size);
  if (l.stream) {
    W4StreamParams p{};
    p.w = w;
    p.X = reinterpret_cast<const uint16_t*>(X); p.ldx = ldx;
    p.Y = reinterpret_cast<uint16_t*>(out); p.ldy = N;
    p.bias = reinterpret_cast<const uint16_t*>(bias);
    p.T = M;
    return dtype == MP_BF16 ? run_stream<true>(d, p, stream) : run_stream<false>(d, p, stream);
  }
  return dtype == MP_BF16 ? run_mma<true>(d, l, w, grad, M, X, ldx, inner, bias, out, ws, stream)
                          : run_mma<false>(d, l, w, grad, M, X, ldx, inner, bias, out, ws, stream);
}

}  // namespace

extern "C" {

int mp_w4_pack(int N, int K, const uint8_t* q, long long ldq, uint32_t* packed, void* stream) {
  if (N < 0 || K < 0 || ldq < K || N > kMaxExtent || K > kMaxExtent)
    return host_fail(MP_ERR_INVALID_ARG, "mp_w4_pack: needs N >= 0, K >= 0, neither above 2^28, ldq >= K");
  if (N == 0 || K == 0) return MP_OK;
  if (q == nullptr || packed == nullptr) return host_fail(MP_ERR_INVALID_ARG, "mp_w4_pack: null pointer");
  HostDevice d;
  if (int rc = host_device(&d)) return rc;
  const int blocks = ceil_div(K, 128);
  const long long words = (long long)N * blocks * 16;
  w4_pack_kernel<<<(unsigned)std::min<long long>((words + 255) / 256, d.sms * 16), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      q, ldq, packed, N, K, blocks);
  MP_HOST_CUDA_TRY(cudaGetLastError());
  host_count_launches(1);
  return MP_OK;
}

int mp_linear_w4_workspace(int M, int N, int K, int group_size, const void* X, long long ldx, int grad_input, size_t* bytes) {
  if (bytes == nullptr) return host_fail(MP_ERR_INVALID_ARG, "mp_linear_w4_workspace: null pointer");
  if (int rc = check_shape("mp_linear_w4_workspace", M, N, K, group_size)) return rc;
  *bytes = M == 0 ? 0 : w4_plan(M, N, K, group_size, grad_input != 0, !tokens_aligned(X, ldx)).total;
  return MP_OK;
}

int mp_debug_w4_launch(int M, int N, int K, int group_size, int grad_input, int out[8]) {
  if (out == nullptr || M == 0) return host_fail(MP_ERR_INVALID_ARG, "mp_debug_w4_launch: needs M > 0 and a result pointer");
  if (int rc = check_shape("mp_debug_w4_launch", M, N, K, group_size)) return rc;
  const Plan l = w4_plan(M, N, K, group_size, grad_input != 0, false);
  const int v[8] = {l.stream, l.bn, l.tiles_m * l.tiles_n * l.split, l.split, l.steps, l.steps_per_split, l.stages, l.raw_slots};
  std::copy(v, v + 8, out);
  return MP_OK;
}

int mp_linear_w4(int dtype, int M, int N, int K, const void* X, long long ldx, const uint32_t* packed, const void* scales,
                 const uint8_t* zeros, int group_size, const void* bias, void* Y, void* workspace, size_t workspace_bytes, void* stream) {
  return run_w4("mp_linear_w4", false, dtype, M, N, K, X, ldx, packed, scales, zeros, group_size, bias, Y, workspace, workspace_bytes, stream);
}

int mp_linear_w4_grad_input(int dtype, int M, int N, int K, const void* dY, long long lddy, const uint32_t* packed, const void* scales,
                            const uint8_t* zeros, int group_size, void* dX, void* workspace, size_t workspace_bytes, void* stream) {
  return run_w4("mp_linear_w4_grad_input", true, dtype, M, N, K, dY, lddy, packed, scales, zeros, group_size, nullptr, dX, workspace,
                workspace_bytes, stream);
}

}  // extern "C"
