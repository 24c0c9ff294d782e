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
// The rows live in registers between the passes.
#include <algorithm>

#include "common.cuh"

namespace b200 {
namespace {

enum Activation { kIdentity = 0, kTanh = 1, kSigmoid = 2 };

// One load: a 128-bit word of T, or one element where width, strides or pointers do not allow words.
template <typename T, bool VEC>
struct Word;
template <typename T>
struct Word<T, true> {
  static constexpr int N = Num<T>::kVec;
  using Raw = uint4;
  static __device__ __forceinline__ Raw zero() { return make_uint4(0, 0, 0, 0); }
  static __device__ __forceinline__ Raw load(const T* p) { return ld_stream(p); }
  static __device__ __forceinline__ Raw load_shared_by_rows(const T* p) { return ld_kept(p); }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[N]) { Num<T>::unpack(r, f); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[N]) { st_stream(p, Num<T>::pack(f)); }
};
template <typename T>
struct Word<T, false> {
  static constexpr int N = 1;
  using Raw = T;
  static __device__ __forceinline__ Raw zero() { return Num<T>::down(0.f); }
  static __device__ __forceinline__ Raw load(const T* p) { return *p; }
  static __device__ __forceinline__ Raw load_shared_by_rows(const T* p) { return *p; }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[1]) { f[0] = Num<T>::up(r); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[1]) { *p = Num<T>::down(f[0]); }
};

__device__ __forceinline__ float activate(float g, int act) {
  if (act == kTanh) return tanhf(g);
  if (act == kSigmoid) return __fdiv_rn(1.f, __fadd_rn(1.f, expf(-g)));
  return g;
}
// d act / d g from the activation's value
__device__ __forceinline__ float activation_slope(float value, int act) {
  if (act == kTanh) return __fsub_rn(1.f, __fmul_rn(value, value));
  if (act == kSigmoid) return __fmul_rn(value, __fsub_rn(1.f, value));
  return 1.f;
}

__device__ __forceinline__ float inv_rms(float sumsq, float cols, float eps) {
  return __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(sumsq, cols), eps)));
}

// N sums over the TPR threads of a row.  TPR <= 32: shuffles.  Wider: the row owns the CTA; one barrier, `slot` is
// shared memory that no thread still reads from an earlier call.
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*slot)[32]) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = __fadd_rn(v[n], __shfl_xor_sync(0xffffffffu, v[n], o));
  }
  if constexpr (TPR > 32) {
    constexpr int WARPS = TPR / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) slot[n][warp] = v[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = slot[n][lane & (WARPS - 1)];
#pragma unroll
      for (int o = WARPS / 2; o > 0; o >>= 1) v[n] = __fadd_rn(v[n], __shfl_xor_sync(0xffffffffu, v[n], o));
    }
  }
}

template <typename T>
struct ForwardArgs {
  const T *x, *residual, *weight, *post, *gate;
  T *y, *s;
  float2* stats;
  uint32_t rows, period;  // period: consecutive rows that share a gate row
  int words;              // loads per row
  int64_t ldx, ldr, ldgate, ldy, lds;
  float cols, eps, offset, scale, residual_scale;
  int act;
};

// One row per TPR threads, ITEMS loads per thread, the row in registers: x and residual as loaded, then s in fp32.
template <typename T, bool VEC, int TPR, int ITEMS>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR)
gated_add_rms_kernel(const ForwardArgs<T> a) {
  using W = Word<T, VEC>;
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
    float sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      float f[N];
      W::unpack(xv[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) sum[0] = __fmaf_rn(f[j], f[j], sum[0]);
    }
    row_sums<TPR, 1>(sum, &slots[0]);
    r1 = inv_rms(sum[0], a.cols, a.eps);
  }
  const T* gr = a.gate == nullptr ? nullptr : a.gate + (live ? row / a.period : 0) * a.ldgate;
  float s[ITEMS][N];
  float sum[1] = {0.f};
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
      for (int j = 0; j < N; ++j) f[j] *= activate(g[j], a.act);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      s[i][j] = fmaf(a.scale, f[j], a.residual_scale * s[i][j]);
      sum[0] = __fmaf_rn(s[i][j], s[i][j], sum[0]);
    }
    if (ok[i]) W::store(a.s + row * a.lds + c, s[i]);
  }
  row_sums<TPR, 1>(sum, &slots[1]);
  const float r2 = inv_rms(sum[0], a.cols, a.eps);
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

// s of one element, for the kernels that go over a row more than once
template <typename T>
__device__ __forceinline__ float stream_value(float x, float residual, float factor, float r1, float residual_scale) {
  return fmaf(r1 * factor, x, residual_scale * residual);
}
// scale * act(gate) * (post_weight + offset) of one column
template <typename T>
__device__ __forceinline__ float branch_factor(const T* post, const T* gate_row, int64_t c, float offset, float scale, int act) {
  float f = scale;
  if (gate_row != nullptr) f *= activate(Num<T>::up(gate_row[c]), act);
  if (post != nullptr) f *= Num<T>::up(post[c]) + offset;
  return f;
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
    float sum[1] = {0.f};
    for (int64_t c = threadIdx.x; c < cols; c += 512) {
      const float f = Num<T>::up(xr[c]);
      sum[0] = __fmaf_rn(f, f, sum[0]);
    }
    row_sums<512, 1>(sum, &slots[0]);
    r1 = inv_rms(sum[0], a.cols, a.eps);
  }
  float sum[1] = {0.f};
  for (int64_t c = threadIdx.x; c < cols; c += 512) {
    const float f = branch_factor(a.post, gr, c, a.offset, a.scale, a.act);
    const float s = stream_value<T>(Num<T>::up(xr[c]), Num<T>::up(rr[c]), f, r1, a.residual_scale);
    sum[0] = __fmaf_rn(s, s, sum[0]);
  }
  row_sums<512, 1>(sum, &slots[1]);
  const float r2 = inv_rms(sum[0], a.cols, a.eps);
  if (a.stats != nullptr && threadIdx.x == 0) a.stats[row] = make_float2(r1, r2);
  for (int64_t c = threadIdx.x; c < cols; c += 512) {
    const float f = branch_factor(a.post, gr, c, a.offset, a.scale, a.act);
    const float s = stream_value<T>(Num<T>::up(xr[c]), Num<T>::up(rr[c]), f, r1, a.residual_scale);
    a.s[row * a.lds + c] = Num<T>::down(s);
    a.y[row * a.ldy + c] = Num<T>::down(s * r2 * (Num<T>::up(a.weight[c]) + a.offset));
  }
}

template <typename T, bool VEC, int TPR, int ITEMS>
int launch_forward(const ForwardArgs<T>& a, cudaStream_t st) {
  constexpr int ROWS = TPR < 128 ? 128 / TPR : 1;
  launch(gated_add_rms_kernel<T, VEC, TPR, ITEMS>, static_cast<unsigned>(ceil_div(a.rows, ROWS)), TPR < 128 ? 128 : TPR, 0, st, a);
  return after_launch("gated_add_rms_kernel");
}

template <typename T>
int run_forward(ForwardArgs<T> a, int64_t cols, bool vec, cudaStream_t st) {
  constexpr int V = Num<T>::kVec;
  if (vec && cols <= 4096 * V) {
    a.words = static_cast<int>(cols / V);
    if (a.words <= 32) return launch_forward<T, true, 32, 1>(a, st);
    if (a.words <= 64) return launch_forward<T, true, 32, 2>(a, st);
    if (a.words <= 128) return launch_forward<T, true, 32, 4>(a, st);
    if (a.words <= 256) return launch_forward<T, true, 128, 2>(a, st);
    if (a.words <= 512) return launch_forward<T, true, 256, 2>(a, st);
    if (a.words <= 1024) return launch_forward<T, true, 256, 4>(a, st);
    if (a.words <= 2048) return launch_forward<T, true, 512, 4>(a, st);
    return launch_forward<T, true, 1024, 4>(a, st);
  }
  if (cols <= 16384) {
    a.words = static_cast<int>(cols);
    if (cols <= 256) return launch_forward<T, false, 32, 8>(a, st);
    if (cols <= 2048) return launch_forward<T, false, 256, 8>(a, st);
    if (cols <= 8192) return launch_forward<T, false, 512, 16>(a, st);
    return launch_forward<T, false, 1024, 16>(a, st);
  }
  launch(gated_add_rms_wide_kernel<T>, a.rows, 512, 0, st, a, cols);
  return after_launch("gated_add_rms_wide_kernel");
}

// ---------------------------------------------------------------- backward --
//
// With a = scale act(gate), f = a (post_weight + offset), s = residual_scale residual + r1 f x and gw = gy (weight + offset):
//   ds = gs + r2 gw - c2 s,       c2 = r2^3 <gw, s> / cols
//   grad_residual = residual_scale ds
//   grad_x = r1 f ds - c1 x,      c1 = r1^3 <f ds, x> / cols    (no c1 without post_weight)
//   <f ds, x> = <f x, gs> + r2 <f x, gw> - c2 <f x, s>: all four sums come from one pass over the row, one barrier.
//   grad_weight = sum over rows of gy s r2
//   k = ds x r1 summed over the rows that share a gate row gives both other gradients:
//   grad_gate = scale act'(gate) (post_weight + offset) k,  grad_post_weight = sum over gate rows of a k
//   A gate of its own for each row has its gradient written with the row, and a k is summed instead of k.
//
// Each walker (a CTA, or a warp for narrow rows) goes over a contiguous range of rows with the sums of its columns in
// registers, and writes a line of them to scratch at its end; with several gate rows also a line of k whenever the
// gate row changes, at index walker + gate row, which no other pair (walker, gate row) has.  gated_columns_kernel adds
// the lines up in a fixed order: the result does not depend on timing.
constexpr int kBackwardThreads = 256;

template <typename T>
struct BackwardArgs {
  const T *gy, *gs, *x, *residual, *weight, *post, *gate;
  const float2* stats;
  T *dx, *dresidual, *dgate;
  float *weight_lines, *branch_lines;
  uint32_t rows, period;
  int words, walkers;
  bool by_group;  // several gate rows, each shared by several rows
  int64_t ldgy, ldgs, ldx, ldr, ldgate, ldo;
  float cols, offset, scale, residual_scale;
  int act;
};

__device__ __forceinline__ uint32_t range_start(uint32_t rows, int walkers, int walker) {
  return static_cast<uint32_t>(static_cast<uint64_t>(rows) * walker / walkers);
}

template <typename T, bool VEC, int TPR, int ITEMS, bool ROW_GATE>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
gated_backward_kernel(const BackwardArgs<T> a) {
  using W = Word<T, VEC>;
  constexpr int N = W::N;
  constexpr int THREADS = TPR < 256 ? 256 : TPR;
  constexpr int GROUPS = THREADS / TPR;
  pdl_prologue();
  __shared__ float slots[2][4][32];
  const int lane_in_row = threadIdx.x % TPR;
  const int walker = blockIdx.x * GROUPS + threadIdx.x / TPR;
  const int64_t cols = static_cast<int64_t>(a.words) * N;
  bool ok[ITEMS];
  float factor[ITEMS][N], sum_w[ITEMS][N], sum_k[ITEMS][N];
  typename W::Raw wv[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int w = lane_in_row + i * TPR;
    ok[i] = w < a.words;
    wv[i] = ok[i] ? W::load_shared_by_rows(a.weight + w * N) : W::zero();
#pragma unroll
    for (int j = 0; j < N; ++j) sum_w[i][j] = sum_k[i][j] = 0.f;
  }
  // f of this thread's columns; without the gate where every row has its own
  auto load_factor = [&](uint32_t gate_row) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int64_t c = static_cast<int64_t>(lane_in_row + i * TPR) * N;
#pragma unroll
      for (int j = 0; j < N; ++j)
        factor[i][j] = ok[i] ? branch_factor<T>(a.post, ROW_GATE || a.gate == nullptr ? nullptr : a.gate + gate_row * a.ldgate, c + j, a.offset, a.scale, a.act) : 0.f;
    }
  };
  auto write_line = [&](float* line, float (&sums)[ITEMS][N]) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (!ok[i]) continue;
      const int64_t c = static_cast<int64_t>(lane_in_row + i * TPR) * N;
#pragma unroll
      for (int j = 0; j < N; ++j) line[c + j] = sums[i][j];
    }
  };
  const uint32_t first = range_start(a.rows, a.walkers, walker), last = walker < a.walkers ? range_start(a.rows, a.walkers, walker + 1) : first;
  uint32_t gate_row = 0, gate_end = a.rows;  // rows below gate_end share gate_row
  if (!ROW_GATE && a.gate != nullptr && first < last) {
    gate_row = first / a.period;
    gate_end = (gate_row + 1) * a.period;
  }
  load_factor(gate_row);
  int parity = 0;
  for (uint32_t row = first; row < last; ++row, parity ^= 1) {
    if (!ROW_GATE && row >= gate_end) {
      write_line(a.branch_lines + static_cast<int64_t>(walker + gate_row) * cols, sum_k);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) sum_k[i][j] = 0.f;
      ++gate_row;
      gate_end += a.period;
      load_factor(gate_row);
    }
    typename W::Raw xv[ITEMS], rv[ITEMS], gyv[ITEMS], gsv[ITEMS], gv[ROW_GATE ? ITEMS : 1];
    const float2 stat = a.stats[row];
    const float r1 = stat.x, r2 = stat.y;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      xv[i] = rv[i] = gyv[i] = gsv[i] = W::zero();
      if constexpr (ROW_GATE) gv[i] = W::zero();
      if (ok[i]) {
        const int c = (lane_in_row + i * TPR) * N;
        xv[i] = W::load(a.x + row * a.ldx + c);
        rv[i] = W::load(a.residual + row * a.ldr + c);
        gyv[i] = W::load(a.gy + row * a.ldgy + c);
        if (a.gs != nullptr) gsv[i] = W::load(a.gs + row * a.ldgs + c);
        if constexpr (ROW_GATE) gv[i] = W::load(a.gate + row * a.ldgate + c);
      }
    }
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      float x[N], r[N], gy[N], gs[N], w[N], g[N];
      W::unpack(xv[i], x);
      W::unpack(rv[i], r);
      W::unpack(gyv[i], gy);
      W::unpack(gsv[i], gs);
      W::unpack(wv[i], w);
      if constexpr (ROW_GATE) W::unpack(gv[i], g);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float f = factor[i][j];
        if constexpr (ROW_GATE) f *= activate(g[j], a.act);
        const float u = f * x[j];
        const float s = stream_value<T>(x[j], r[j], f, r1, a.residual_scale);
        const float gw = gy[j] * (w[j] + a.offset);
        sums[0] = fmaf(gw, s, sums[0]);
        sums[1] = fmaf(u, gs[j], sums[1]);
        sums[2] = fmaf(u, gw, sums[2]);
        sums[3] = fmaf(u, s, sums[3]);
      }
    }
    row_sums<TPR, 4>(sums, slots[parity]);
    const float c2 = r2 * r2 * r2 * __fdiv_rn(sums[0], a.cols);
    const float inner = sums[1] + r2 * sums[2] - c2 * sums[3];
    const float c1 = a.post == nullptr ? 0.f : r1 * r1 * r1 * __fdiv_rn(inner, a.cols);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (!ok[i]) continue;
      const int64_t c = static_cast<int64_t>(lane_in_row + i * TPR) * N;
      float x[N], r[N], gy[N], gs[N], w[N], g[N], dx[N];
      W::unpack(xv[i], x);
      W::unpack(rv[i], r);
      W::unpack(gyv[i], gy);
      W::unpack(gsv[i], gs);
      W::unpack(wv[i], w);
      if constexpr (ROW_GATE) W::unpack(gv[i], g);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float f = factor[i][j], value = 1.f;
        if constexpr (ROW_GATE) {
          value = activate(g[j], a.act);
          f *= value;
        }
        const float s = stream_value<T>(x[j], r[j], f, r1, a.residual_scale);
        const float ds = fmaf(-c2, s, fmaf(r2, gy[j] * (w[j] + a.offset), gs[j]));
        const float k = ds * x[j] * r1;
        dx[j] = fmaf(r1 * f, ds, -c1 * x[j]);
        r[j] = a.residual_scale * ds;
        sum_w[i][j] = fmaf(gy[j] * r2, s, sum_w[i][j]);
        if constexpr (ROW_GATE) {
          sum_k[i][j] = fmaf(a.scale * value, k, sum_k[i][j]);
          g[j] = factor[i][j] * activation_slope(value, a.act) * k;
        } else {
          sum_k[i][j] += k;
        }
      }
      W::store(a.dx + row * a.ldo + c, dx);
      W::store(a.dresidual + row * a.ldo + c, r);
      if constexpr (ROW_GATE) W::store(a.dgate + row * a.ldo + c, g);
    }
  }
  if (walker >= a.walkers) return;
  write_line(a.weight_lines + walker * cols, sum_w);
  if (a.branch_lines != nullptr && (!a.by_group || first < last)) write_line(a.branch_lines + static_cast<int64_t>(walker + gate_row) * cols, sum_k);
}

// Any width: one CTA per walker, the row read twice, the sums of a walker's columns kept in its lines in scratch.
template <typename T>
__global__ void __launch_bounds__(kBackwardThreads)
gated_backward_wide_kernel(const BackwardArgs<T> a, int64_t cols, bool row_gate) {
  pdl_prologue();
  __shared__ float slots[2][4][32];
  const int walker = blockIdx.x;
  const uint32_t first = range_start(a.rows, a.walkers, walker), last = range_start(a.rows, a.walkers, walker + 1);
  float* sum_w = a.weight_lines + walker * cols;
  const bool shared_gate = a.gate != nullptr && !row_gate;
  uint32_t gate_row = shared_gate ? first / a.period : 0;
  float* sum_k = a.branch_lines == nullptr ? nullptr : a.branch_lines + static_cast<int64_t>(walker + gate_row) * cols;
  // a thread only ever touches its own columns of a line: no barrier is needed between these and the sums below
  for (int64_t c = threadIdx.x; c < cols; c += kBackwardThreads) sum_w[c] = 0.f;
  auto clear_k = [&] {
    if (sum_k != nullptr)
      for (int64_t c = threadIdx.x; c < cols; c += kBackwardThreads) sum_k[c] = 0.f;
  };
  if (!a.by_group || first < last) clear_k();
  int parity = 0;
  for (uint32_t row = first; row < last; ++row, parity ^= 1) {
    if (shared_gate && row / a.period != gate_row) {
      gate_row = row / a.period;
      sum_k = a.branch_lines + static_cast<int64_t>(walker + gate_row) * cols;
      clear_k();
    }
    const float2 stat = a.stats[row];
    const float r1 = stat.x, r2 = stat.y;
    const T *xr = a.x + row * a.ldx, *rr = a.residual + row * a.ldr, *gyr = a.gy + row * a.ldgy;
    const T* gsr = a.gs == nullptr ? nullptr : a.gs + row * a.ldgs;
    const T* gr = a.gate == nullptr ? nullptr : a.gate + (row_gate ? row : gate_row) * a.ldgate;
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t c = threadIdx.x; c < cols; c += kBackwardThreads) {
      const float f = branch_factor(a.post, gr, c, a.offset, a.scale, a.act), x = Num<T>::up(xr[c]);
      const float s = stream_value<T>(x, Num<T>::up(rr[c]), f, r1, a.residual_scale);
      const float gw = Num<T>::up(gyr[c]) * (Num<T>::up(a.weight[c]) + a.offset), u = f * x;
      sums[0] = fmaf(gw, s, sums[0]);
      if (gsr != nullptr) sums[1] = fmaf(u, Num<T>::up(gsr[c]), sums[1]);
      sums[2] = fmaf(u, gw, sums[2]);
      sums[3] = fmaf(u, s, sums[3]);
    }
    row_sums<kBackwardThreads, 4>(sums, slots[parity]);
    const float c2 = r2 * r2 * r2 * __fdiv_rn(sums[0], a.cols);
    const float inner = sums[1] + r2 * sums[2] - c2 * sums[3];
    const float c1 = a.post == nullptr ? 0.f : r1 * r1 * r1 * __fdiv_rn(inner, a.cols);
    for (int64_t c = threadIdx.x; c < cols; c += kBackwardThreads) {
      const float p = a.post == nullptr ? 1.f : Num<T>::up(a.post[c]) + a.offset;
      const float value = gr == nullptr ? 1.f : activate(Num<T>::up(gr[c]), a.act);
      const float branch = a.scale * value, f = branch * p, x = Num<T>::up(xr[c]), gy = Num<T>::up(gyr[c]);
      const float s = stream_value<T>(x, Num<T>::up(rr[c]), f, r1, a.residual_scale);
      const float ds = fmaf(-c2, s, fmaf(r2, gy * (Num<T>::up(a.weight[c]) + a.offset), gsr == nullptr ? 0.f : Num<T>::up(gsr[c])));
      const float k = ds * x * r1;
      a.dx[row * a.ldo + c] = Num<T>::down(fmaf(r1 * f, ds, -c1 * x));
      a.dresidual[row * a.ldo + c] = Num<T>::down(a.residual_scale * ds);
      sum_w[c] = fmaf(gy * r2, s, sum_w[c]);
      if (sum_k != nullptr) sum_k[c] += row_gate ? branch * k : k;
      if (row_gate) a.dgate[row * a.ldo + c] = Num<T>::down(a.scale * p * activation_slope(value, a.act) * k);
    }
  }
}

// Adds the walkers' lines up: grad_weight from weight_lines, and from branch_lines grad_post_weight and the gradient of
// a gate that rows share.  A CTA owns 32 columns; its eight warps take every eighth line (or gate row) each, then the
// eight sums are added in warp order.
template <typename T>
struct ColumnArgs {
  const float *weight_lines, *branch_lines;
  const T *post, *gate;
  T *dweight, *dpost, *dgate;
  int64_t cols, ldgate;
  uint32_t rows, period;
  int weight_count, walkers, gate_rows;  // gate_rows: 0 unless rows share gate rows
  float offset, scale, line_scale;  // line_scale: what a sum over branch_lines lacks of grad_post_weight
  int act;
};
template <typename T>
__global__ void __launch_bounds__(256)
gated_columns_kernel(const ColumnArgs<T> a) {
  pdl_prologue();
  __shared__ float part[2][8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sum_w = 0.f, sum_p = 0.f;
  if (c < a.cols) {
#pragma unroll 4
    for (int l = warp; l < a.weight_count; l += 8) sum_w += a.weight_lines[l * a.cols + c];
    if (a.branch_lines != nullptr && a.gate_rows <= 1) {
#pragma unroll 4
      for (int l = warp; l < a.weight_count; l += 8) sum_p += a.branch_lines[l * a.cols + c];
    } else if (a.branch_lines != nullptr) {
      const float p = a.post == nullptr ? 1.f : Num<T>::up(a.post[c]) + a.offset;
      for (int g = warp; g < a.gate_rows; g += 8) {
        // walkers whose rows meet this gate row's: those from the one that holds its first row to the one that holds its last
        const uint64_t lo = static_cast<uint64_t>(g) * a.period, hi = lo + a.period;
        int w = a.rows == 0 ? 0 : static_cast<int>(lo * a.walkers / a.rows);
        while (w > 0 && range_start(a.rows, a.walkers, w) > lo) --w;
        while (w + 1 < a.walkers && range_start(a.rows, a.walkers, w + 1) <= lo) ++w;
        float k = 0.f;
        for (; w < a.walkers && range_start(a.rows, a.walkers, w) < hi; ++w)
          if (range_start(a.rows, a.walkers, w + 1) > range_start(a.rows, a.walkers, w)) k += a.branch_lines[static_cast<int64_t>(w + g) * a.cols + c];
        const float value = activate(Num<T>::up(a.gate[g * a.ldgate + c]), a.act);
        a.dgate[g * a.cols + c] = Num<T>::down(a.scale * p * activation_slope(value, a.act) * k);
        sum_p += a.scale * value * k;
      }
    }
  }
  part[0][warp][lane] = sum_w;
  part[1][warp][lane] = sum_p;
  __syncthreads();
  if (warp == 0 && c < a.cols) {
    sum_w = sum_p = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      sum_w += part[0][k][lane];
      sum_p += part[1][k][lane];
    }
    a.dweight[c] = Num<T>::down(sum_w);
    if (a.gate_rows == 1) {
      const float value = activate(Num<T>::up(a.gate[c]), a.act), p = a.post == nullptr ? 1.f : Num<T>::up(a.post[c]) + a.offset;
      a.dgate[c] = Num<T>::down(a.scale * p * activation_slope(value, a.act) * sum_p);
      sum_p *= a.scale * value;
    }
    if (a.dpost != nullptr) a.dpost[c] = Num<T>::down(a.line_scale * sum_p);
  }
}

// How many walkers share the rows, and the threads of a walker.
struct BackwardPlan {
  bool vec, wide;
  int tpr;
  int walkers;
};
BackwardPlan plan_backward(int64_t rows, int64_t cols, int dtype, bool aligned_rows) {
  BackwardPlan p;
  const int64_t v = dtype == B200_F32 ? 4 : 8;
  p.vec = aligned_rows && cols % v == 0;
  const int64_t words = p.vec ? cols / v : cols;
  const int64_t narrow = p.vec ? 128 : 512, limit = p.vec ? 1024 : 4096;
  p.wide = words > limit;
  p.tpr = words <= narrow ? 32 : words <= limit / 2 || p.wide ? 256 : 512;
  const int64_t ctas = static_cast<int64_t>(sm_count()) * (p.tpr == 512 ? 1 : 2);
  const int64_t groups = p.tpr == 32 ? kBackwardThreads / 32 : 1;
  p.walkers = static_cast<int>(std::max<int64_t>(1, std::min(rows, ctas * groups)));
  return p;
}
// Lines of scratch: one of grad_weight for each walker; of k one for each, and one more for each change of the gate row.
int64_t scratch_lines(int64_t walkers, int64_t rows, int64_t gate_rows) {
  return 2 * walkers + (gate_rows > 1 && gate_rows < rows ? gate_rows : 0);
}

template <typename T, bool VEC, int TPR, int ITEMS>
int launch_backward(const BackwardArgs<T>& a, bool row_gate, cudaStream_t st) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR;
  const unsigned grid = static_cast<unsigned>(ceil_div(a.walkers, THREADS / TPR));
  if (row_gate) launch(gated_backward_kernel<T, VEC, TPR, ITEMS, true>, grid, THREADS, 0, st, a);
  else launch(gated_backward_kernel<T, VEC, TPR, ITEMS, false>, grid, THREADS, 0, st, a);
  return after_launch("gated_backward_kernel");
}

template <typename T>
int run_backward(BackwardArgs<T> a, ColumnArgs<T> c, int64_t cols, const BackwardPlan& p, bool row_gate, cudaStream_t st) {
  int rc;
  if (p.wide) {
    launch(gated_backward_wide_kernel<T>, static_cast<unsigned>(a.walkers), kBackwardThreads, 0, st, a, cols, row_gate);
    rc = after_launch("gated_backward_wide_kernel");
  } else if (p.vec) {
    a.words = static_cast<int>(cols / Num<T>::kVec);
    if (a.words <= 32) rc = launch_backward<T, true, 32, 1>(a, row_gate, st);
    else if (p.tpr == 32) rc = launch_backward<T, true, 32, 4>(a, row_gate, st);
    else if (a.words <= 256) rc = launch_backward<T, true, 256, 1>(a, row_gate, st);
    else if (p.tpr == 256) rc = launch_backward<T, true, 256, 2>(a, row_gate, st);
    else rc = launch_backward<T, true, 512, 2>(a, row_gate, st);
  } else {
    a.words = static_cast<int>(cols);
    if (p.tpr == 32) rc = launch_backward<T, false, 32, 16>(a, row_gate, st);
    else if (p.tpr == 256) rc = launch_backward<T, false, 256, 8>(a, row_gate, st);
    else rc = launch_backward<T, false, 512, 8>(a, row_gate, st);
  }
  if (rc) return rc;
  launch(gated_columns_kernel<T>, static_cast<unsigned>(ceil_div(cols, 32)), 256, 0, st, c);
  return after_launch("gated_columns_kernel");
}

// Sizes and enums that both directions check alike.
int check_shapes(const char* fn, int64_t rows, int64_t cols, int64_t gate_rows, const void* gate, int dtype, int activation) {
  if (!dtype_ok(dtype)) return fail(B200_ERR_DTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (activation < kIdentity || activation > kSigmoid) return fail(B200_ERR_SHAPE, "%s: unknown activation %d", fn, activation);
  if (rows < 0 || cols < 0 || gate_rows < 0) return fail(B200_ERR_SHAPE, "%s: negative size (rows=%lld, cols=%lld, gate_rows=%lld)", fn, (long long)rows, (long long)cols, (long long)gate_rows);
  if (rows > 0x7fffffffLL || cols > 0x7fffffffLL) return fail(B200_ERR_SHAPE, "%s: rows=%lld and cols=%lld must be below 2^31", fn, (long long)rows, (long long)cols);
  if (rows > 0 && gate != nullptr && (gate_rows == 0 || rows % gate_rows != 0))
    return fail(B200_ERR_SHAPE, "%s: rows=%lld is not a multiple of gate_rows=%lld", fn, (long long)rows, (long long)gate_rows);
  return B200_OK;
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
  const int64_t v = 16 / static_cast<int64_t>(es);
  const bool vec = cols % v == 0 && ldx % v == 0 && ldr % v == 0 && ldy % v == 0 && lds % v == 0 && aligned(x, 16) && aligned(residual, 16) &&
                   aligned(weight, 16) && aligned(post_weight, 16) && aligned(y, 16) && aligned(s, 16) &&
                   (gate == nullptr || (aligned(gate, 16) && (gate_rows == 1 || ldgate % v == 0)));
  B200_DISPATCH_DTYPE(dtype, T, {
    ForwardArgs<T> a;
    a.x = static_cast<const T*>(x), a.residual = static_cast<const T*>(residual), a.weight = static_cast<const T*>(weight);
    a.post = static_cast<const T*>(post_weight), a.gate = static_cast<const T*>(gate);
    a.y = static_cast<T*>(y), a.s = static_cast<T*>(s), a.stats = reinterpret_cast<float2*>(stats);
    a.rows = static_cast<uint32_t>(rows), a.period = gate == nullptr ? 1 : static_cast<uint32_t>(rows / gate_rows);
    a.ldx = ldx, a.ldr = ldr, a.ldgate = ldgate, a.ldy = ldy, a.lds = lds;
    a.cols = static_cast<float>(cols), a.eps = static_cast<float>(eps), a.offset = static_cast<float>(offset);
    a.scale = static_cast<float>(scale), a.residual_scale = static_cast<float>(residual_scale), a.act = activation;
    a.words = 0;
    return run_forward<T>(a, cols, vec, static_cast<cudaStream_t>(stream));
  });
  return B200_OK;
}

extern "C" int b200_gated_add_rms_norm_backward_scratch_bytes(int64_t rows, int64_t cols, int64_t gate_rows, int dtype, size_t* bytes) {
  B200_REQUIRE_PTR(bytes);
  if (int rc = check_shapes(__func__, rows, cols, gate_rows, nullptr, dtype, kIdentity)) return rc;
  if (int rc = check_device()) return rc;
  // the element-wise plan of a width may use more walkers than the word-wise one: take the larger
  const int64_t walkers = std::max(plan_backward(rows, cols, dtype, true).walkers, plan_backward(rows, cols, dtype, false).walkers);
  *bytes = static_cast<size_t>(scratch_lines(walkers, rows, gate_rows)) * static_cast<size_t>(cols) * sizeof(float);
  return B200_OK;
}

extern "C" int b200_gated_add_rms_norm_backward(const void* grad_y, const void* grad_s, const void* x, const void* residual, const void* weight,
                                                const void* post_weight, const void* gate, const float* stats, void* grad_x, void* grad_residual,
                                                void* grad_weight, void* grad_post_weight, void* grad_gate, int64_t rows, int64_t cols,
                                                int64_t gate_rows, int64_t ldgy, int64_t ldgs, int64_t ldx, int64_t ldr, int64_t ldgate, int dtype,
                                                int activation, double scale, double residual_scale, double offset, void* scratch,
                                                size_t scratch_bytes, void* stream) {
  if (int rc = check_shapes(__func__, rows, cols, gate_rows, gate, dtype, activation)) return rc;
  if (cols == 0) return B200_OK;
  B200_REQUIRE_PTR(weight);
  B200_REQUIRE_PTR(grad_weight);
  if (rows > 0) {
    B200_REQUIRE_PTR(scratch);
    B200_REQUIRE_PTR(grad_y);
    B200_REQUIRE_PTR(x);
    B200_REQUIRE_PTR(residual);
    B200_REQUIRE_PTR(stats);
    B200_REQUIRE_PTR(grad_x);
    B200_REQUIRE_PTR(grad_residual);
    if (ldgy < cols || (grad_s && ldgs < cols) || ldx < cols || ldr < cols || (gate && gate_rows > 1 && ldgate < cols))
      return fail(B200_ERR_SHAPE, "%s: leading dimension smaller than cols", __func__);
  }
  if ((post_weight == nullptr) != (grad_post_weight == nullptr) || ((gate == nullptr) != (grad_gate == nullptr)))
    return fail(B200_ERR_NULL_POINTER, "%s: post_weight and grad_post_weight, gate and grad_gate go together", __func__);
  const size_t es = dtype_size(dtype);
  const void* all[] = {grad_y, grad_s, x, residual, weight, post_weight, gate, grad_x, grad_residual, grad_weight, grad_post_weight, grad_gate};
  bool words = true;
  for (const void* p : all) {
    if (!aligned(p, es)) return fail(B200_ERR_ALIGNMENT, "%s: pointer not aligned to the element size", __func__);
    words = words && aligned(p, 16);
  }
  if (!aligned(stats, 8)) return fail(B200_ERR_ALIGNMENT, "%s: stats must be 8-byte aligned", __func__);
  if (int rc = check_device()) return rc;
  if (rows == 0) {
    if (cudaMemsetAsync(grad_weight, 0, cols * es, static_cast<cudaStream_t>(stream)) != cudaSuccess ||
        (grad_post_weight && cudaMemsetAsync(grad_post_weight, 0, cols * es, static_cast<cudaStream_t>(stream)) != cudaSuccess) ||
        (grad_gate && cudaMemsetAsync(grad_gate, 0, gate_rows * cols * es, static_cast<cudaStream_t>(stream)) != cudaSuccess))
      return fail(B200_ERR_LAUNCH, "%s: %s", __func__, cudaGetErrorString(cudaGetLastError()));
    return B200_OK;
  }
  const int64_t v = 16 / static_cast<int64_t>(es);
  words = words && ldgy % v == 0 && (grad_s == nullptr || ldgs % v == 0) && ldx % v == 0 && ldr % v == 0 &&
          (gate == nullptr || gate_rows <= 1 || ldgate % v == 0);
  const BackwardPlan p = plan_backward(rows, cols, dtype, words);
  const size_t need = static_cast<size_t>(scratch_lines(p.walkers, rows, gate_rows)) * static_cast<size_t>(cols) * sizeof(float);
  if (scratch_bytes < need || !aligned(scratch, 16))
    return fail(B200_ERR_SCRATCH, "%s: scratch needs %zu bytes, 16-byte aligned (got %zu)", __func__, need, scratch_bytes);
  const bool row_gate = gate != nullptr && gate_rows == rows && rows > 1;
  const bool shared_gate = gate != nullptr && !row_gate;
  B200_DISPATCH_DTYPE(dtype, T, {
    BackwardArgs<T> a;
    a.gy = static_cast<const T*>(grad_y), a.gs = static_cast<const T*>(grad_s), a.x = static_cast<const T*>(x);
    a.residual = static_cast<const T*>(residual), a.weight = static_cast<const T*>(weight), a.post = static_cast<const T*>(post_weight);
    a.gate = static_cast<const T*>(gate), a.stats = reinterpret_cast<const float2*>(stats);
    a.dx = static_cast<T*>(grad_x), a.dresidual = static_cast<T*>(grad_residual), a.dgate = static_cast<T*>(grad_gate);
    a.weight_lines = static_cast<float*>(scratch);
    a.branch_lines = post_weight == nullptr && !shared_gate ? nullptr : a.weight_lines + static_cast<int64_t>(p.walkers) * cols;
    a.rows = static_cast<uint32_t>(rows), a.period = shared_gate ? static_cast<uint32_t>(rows / gate_rows) : 1;
    a.words = 0, a.walkers = p.walkers, a.by_group = shared_gate && gate_rows > 1;
    a.ldgy = ldgy, a.ldgs = ldgs, a.ldx = ldx, a.ldr = ldr, a.ldgate = ldgate, a.ldo = cols;
    a.cols = static_cast<float>(cols), a.offset = static_cast<float>(offset), a.scale = static_cast<float>(scale);
    a.residual_scale = static_cast<float>(residual_scale), a.act = activation;
    ColumnArgs<T> c;
    c.weight_lines = a.weight_lines, c.branch_lines = a.branch_lines, c.post = a.post, c.gate = a.gate;
    c.dweight = static_cast<T*>(grad_weight), c.dpost = static_cast<T*>(grad_post_weight), c.dgate = a.dgate;
    c.cols = cols, c.ldgate = ldgate, c.rows = a.rows, c.period = a.period;
    c.weight_count = p.walkers, c.walkers = p.walkers, c.gate_rows = shared_gate ? static_cast<int>(gate_rows) : 0;
    c.offset = a.offset, c.scale = a.scale, c.line_scale = gate == nullptr ? a.scale : 1.f, c.act = activation;
    return run_backward<T>(a, c, cols, p, row_gate, static_cast<cudaStream_t>(stream));
  });
  return B200_OK;
}
