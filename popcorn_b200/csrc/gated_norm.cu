// The norm that joins a block to the residual stream: an optional RMSNorm of the block's output, its gate and scale,
// the scaled residual add and the RMSNorm in front of the next block, forward and backward.
//
//   n = x r1 (post_weight + offset),  r1 = 1 / sqrt(mean(x^2) + eps)        (n = x without post_weight)
//   s = residual_scale * residual + scale * act(gate) * n
//   y = s r2 (weight + offset),       r2 = 1 / sqrt(mean(s^2) + eps)
//
// Everything is fp32 from the stored words to the one rounding of each output: y is formed from the unrounded s, and
// the backward recomputes s from x and residual, so no rounded intermediate enters a gradient.
//
// Bound: HBM.  Forward: x, residual (and a gate per row) read once, y and s written once.  Backward: x, residual, the
// two incoming gradients read once, two gradients written once (s is not saved: reading residual costs the same).
#include "gated_norm.cuh"

namespace b200 {
namespace {

template <typename T>
struct ForwardArgs {
  const T *x, *residual, *weight, *post, *gate;
  T *y, *s;
  float2* stats;
  uint32_t rows, period;  // period: consecutive rows that share a gate row
  int words;              // loads per row
  int64_t ldx, ldr, ldgate, ldy, lds;
  float inv_cols, eps, offset, scale, residual_scale;
  int act;
};

// One row per TPR threads, ITEMS loads per thread, the row in registers: x and residual as loaded, then s in fp32.
template <typename T, int ACCESS, int TPR, int ITEMS>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR)
gated_add_rms_kernel(const ForwardArgs<T> a) {
  using W = Word<T, ACCESS>;
  constexpr int N = W::N;
  constexpr int THREADS = TPR < 128 ? 128 : TPR;
  pdl_prologue();
  __shared__ float slots[2][32];
  const int lane_in_row = threadIdx.x % TPR;
  const uint32_t row = blockIdx.x * (THREADS / TPR) + threadIdx.x / TPR;
  const bool live = row < a.rows;
  const T* xr = a.x + row * a.ldx;
  const T* rr = a.residual + row * a.ldr;
  typename W::Raw xv[ITEMS], rv[ITEMS];
  bool ok[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int w = lane_in_row + i * TPR;
    ok[i] = live && w < a.words;
    xv[i] = rv[i] = W::zero();
    if (ok[i]) {
      xv[i] = W::load(xr + w * N);
      rv[i] = W::load(rr + w * N);
    }
  }
  float r1 = 1.f;
  if (a.post != nullptr) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      float f[N];
      W::unpack(xv[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) sum = __fmaf_rn(f[j], f[j], sum);
    }
    r1 = inv_rms(row_sum<TPR>(sum, slots[0]), a.inv_cols, a.eps);
  }
  const T* gr = a.gate == nullptr ? nullptr : a.gate + (live ? row / a.period : 0) * a.ldgate;
  float s[ITEMS][N];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = (lane_in_row + i * TPR) * N;
    float f[N];
    W::unpack(xv[i], f);
    W::unpack(rv[i], s[i]);
    if (ok[i] && a.post != nullptr) {
      float p[N];
      W::unpack(W::load_shared_by_rows(a.post + c), p);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = f[j] * r1 * (p[j] + a.offset);
    }
    if (ok[i] && gr != nullptr) {
      float g[N];
      W::unpack(W::load_shared_by_rows(gr + c), g);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] *= activate<T>(g[j], a.act);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      s[i][j] = fmaf(a.scale, f[j], a.residual_scale * s[i][j]);
      sum = __fmaf_rn(s[i][j], s[i][j], sum);
    }
    if (ok[i]) W::store(a.s + row * a.lds + c, s[i]);
  }
  const float r2 = inv_rms(row_sum<TPR>(sum, slots[1]), a.inv_cols, a.eps);
  if (a.stats != nullptr && live && lane_in_row == 0) a.stats[row] = make_float2(r1, r2);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (!ok[i]) continue;
    const int c = (lane_in_row + i * TPR) * N;
    float w[N];
    W::unpack(W::load_shared_by_rows(a.weight + c), w);
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = s[i][j] * r2 * (w[j] + a.offset);
    W::store(a.y + row * a.ldy + c, w);
  }
}

// Rows too wide for registers: one CTA per row, the row read again for each pass (from L2 where it fits).
template <typename T>
__global__ void __launch_bounds__(512)
gated_add_rms_wide_kernel(const ForwardArgs<T> a, int64_t cols) {
  pdl_prologue();
  __shared__ float slots[2][32];
  const int64_t row = blockIdx.x;
  const T *xr = a.x + row * a.ldx, *rr = a.residual + row * a.ldr;
  const T* gr = a.gate == nullptr ? nullptr : a.gate + static_cast<int64_t>(static_cast<uint32_t>(row) / a.period) * a.ldgate;
  float r1 = 1.f;
  if (a.post != nullptr) {
    float sum = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += 512) {
      const float f = Num<T>::up(xr[c]);
      sum = __fmaf_rn(f, f, sum);
    }
    r1 = inv_rms(row_sum<512>(sum, slots[0]), a.inv_cols, a.eps);
  }
  float sum = 0.f;
  for (int64_t c = threadIdx.x; c < cols; c += 512) {
    const float f = branch_factor(a.post, gr, c, a.offset, a.scale, a.act);
    const float s = stream_value(Num<T>::up(xr[c]), Num<T>::up(rr[c]), f, r1, a.residual_scale);
    sum = __fmaf_rn(s, s, sum);
  }
  const float r2 = inv_rms(row_sum<512>(sum, slots[1]), a.inv_cols, a.eps);
  if (a.stats != nullptr && threadIdx.x == 0) a.stats[row] = make_float2(r1, r2);
  for (int64_t c = threadIdx.x; c < cols; c += 512) {
    const float f = branch_factor(a.post, gr, c, a.offset, a.scale, a.act);
    const float s = stream_value(Num<T>::up(xr[c]), Num<T>::up(rr[c]), f, r1, a.residual_scale);
    a.s[row * a.lds + c] = Num<T>::down(s);
    a.y[row * a.ldy + c] = Num<T>::down(s * r2 * (Num<T>::up(a.weight[c]) + a.offset));
  }
}

template <typename T, int ACCESS, int TPR, int ITEMS>
int launch_forward(const ForwardArgs<T>& a, cudaStream_t st) {
  constexpr int ROWS = TPR < 128 ? 128 / TPR : 1;
  launch(gated_add_rms_kernel<T, ACCESS, TPR, ITEMS>, static_cast<unsigned>(ceil_div(a.rows, ROWS)), TPR < 128 ? 128 : TPR, 0, st, a);
  return after_launch("gated_add_rms_kernel");
}

template <typename T>
int run_forward(ForwardArgs<T> a, int64_t cols, Access access, cudaStream_t st) {
  constexpr int V = Num<T>::kVec;
  if (access == kWords && cols <= 4096 * V) {
    a.words = static_cast<int>(cols / V);
    if (a.words <= 32) return launch_forward<T, kWords, 32, 1>(a, st);
    if (a.words <= 64) return launch_forward<T, kWords, 32, 2>(a, st);
    if (a.words <= 128) return launch_forward<T, kWords, 32, 4>(a, st);
    if (a.words <= 256) return launch_forward<T, kWords, 128, 2>(a, st);
    // many rows: more of a row per thread keeps more loads in flight (bf16 [16384, 4096] 92 us with 256 threads, 86 with 128; fp16
    // [16376, 5120] 154 and 135); few rows, where nothing else hides a thread's steps: 4.2 us for eight with 256, 6.2 with 128
    const bool few = a.rows < 4u * static_cast<uint32_t>(sm_count());
    if (few && a.words > 256 && a.words <= 512) return launch_forward<T, kWords, 256, 2>(a, st);
    if (a.words <= 512) return launch_forward<T, kWords, 128, 4>(a, st);
    if (a.words <= 640) return launch_forward<T, kWords, 128, 5>(a, st);
    if (a.words <= 768) return launch_forward<T, kWords, 128, 6>(a, st);
    if (a.words <= 1024) return launch_forward<T, kWords, 256, 4>(a, st);
    if (a.words <= 2048) return launch_forward<T, kWords, 512, 4>(a, st);
    return launch_forward<T, kWords, 1024, 4>(a, st);
  }
  // two elements at a time keep half as many instructions busy for the same bytes ([4095, 2050] fp32 with a gate per row:
  // 47 us, one element at a time 57; [8192, 2050] bf16 64 and 86)
  if (access != kSingles && cols <= 16384) {
    a.words = static_cast<int>(cols / 2);
    if (a.words <= 256) return launch_forward<T, kPairs, 32, 8>(a, st);
    if (a.words <= 1024) return launch_forward<T, kPairs, 128, 8>(a, st);
    if (a.words <= 1536) return launch_forward<T, kPairs, 128, 12>(a, st);
    if (a.words <= 2048) return launch_forward<T, kPairs, 128, 16>(a, st);
    if (a.words <= 4096) return launch_forward<T, kPairs, 256, 16>(a, st);
    return launch_forward<T, kPairs, 512, 16>(a, st);
  }
  if (cols <= 16384) {
    a.words = static_cast<int>(cols);
    if (cols <= 256) return launch_forward<T, kSingles, 32, 8>(a, st);
    if (cols <= 1024) return launch_forward<T, kSingles, 128, 8>(a, st);
    if (cols <= 2048) return launch_forward<T, kSingles, 128, 16>(a, st);
    if (cols <= 4096) return launch_forward<T, kSingles, 256, 16>(a, st);
    if (cols <= 8192) return launch_forward<T, kSingles, 512, 16>(a, st);
    return launch_forward<T, kSingles, 1024, 16>(a, st);
  }
  launch(gated_add_rms_wide_kernel<T>, a.rows, 512, 0, st, a, cols);
  return after_launch("gated_add_rms_wide_kernel");
}

}  // namespace

}  // namespace b200

using namespace b200;

extern "C" int b200_gated_add_rms_norm(const void* x, const void* residual, const void* weight, const void* post_weight, const void* gate,
                                       void* y, void* s, float* stats, int64_t rows, int64_t cols, int64_t gate_rows, int64_t ldx,
                                       int64_t ldr, int64_t ldgate, int64_t ldy, int64_t lds, int dtype, int activation, double scale,
                                       double residual_scale, double eps, double offset, void* stream) {
  if (int rc = check_shapes(__func__, rows, cols, gate_rows, gate, dtype, activation)) return rc;
  if (rows == 0 || cols == 0) return B200_OK;
  B200_REQUIRE_PTR(x);
  B200_REQUIRE_PTR(residual);
  B200_REQUIRE_PTR(weight);
  B200_REQUIRE_PTR(y);
  B200_REQUIRE_PTR(s);
  if (ldx < cols || ldr < cols || ldy < cols || lds < cols || (gate && gate_rows > 1 && ldgate < cols))
    return fail(B200_ERR_SHAPE, "%s: leading dimension smaller than cols", __func__);
  const size_t es = dtype_size(dtype);
  if (!aligned(x, es) || !aligned(residual, es) || !aligned(weight, es) || !aligned(post_weight, es) || !aligned(gate, es) || !aligned(y, es) ||
      !aligned(s, es) || !aligned(stats, 8))
    return fail(B200_ERR_ALIGNMENT, "%s: pointer not aligned to the element size (stats: 8 bytes)", __func__);
  if (int rc = check_device()) return rc;
  const Access access = access_of(es, cols, {x, residual, weight, post_weight, gate, y, s}, {ldx, ldr, ldy, lds, gate != nullptr && gate_rows > 1 ? ldgate : 0});
  B200_DISPATCH_DTYPE(dtype, T, {
    ForwardArgs<T> a;
    a.x = static_cast<const T*>(x), a.residual = static_cast<const T*>(residual), a.weight = static_cast<const T*>(weight);
    a.post = static_cast<const T*>(post_weight), a.gate = static_cast<const T*>(gate);
    a.y = static_cast<T*>(y), a.s = static_cast<T*>(s), a.stats = reinterpret_cast<float2*>(stats);
    a.rows = static_cast<uint32_t>(rows), a.period = gate == nullptr ? 1 : static_cast<uint32_t>(rows / gate_rows);
    a.ldx = ldx, a.ldr = ldr, a.ldgate = ldgate, a.ldy = ldy, a.lds = lds;
    a.inv_cols = 1.f / static_cast<float>(cols), a.eps = static_cast<float>(eps), a.offset = static_cast<float>(offset);
    a.scale = static_cast<float>(scale), a.residual_scale = static_cast<float>(residual_scale), a.act = activation;
    a.words = 0;
    return run_forward<T>(a, cols, access, static_cast<cudaStream_t>(stream));
  });
  return B200_OK;
}
