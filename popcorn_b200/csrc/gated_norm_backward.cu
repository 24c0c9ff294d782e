// Backward of the gated residual norm (gated_norm.cu).
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
// A walker (a CTA of 32 to 512 threads, 16 columns a thread) goes over a contiguous range of rows, which arrive through a
// ring of bulk copies in shared memory, with the sums of its columns in registers, and writes a line of them to scratch at
// its end.  With several gate rows a walker also writes a line of k whenever the gate row
// changes, at index walker + gate row, which no other pair (walker, gate row) has.  gated_columns_kernel adds the lines up
// in a fixed order: the result does not depend on timing.
#include <cstdlib>

#include "gated_norm.cuh"

namespace b200 {
namespace {

constexpr int kBackwardThreads = 256;

template <typename T>
struct BackwardArgs {
  const T *gy, *gs, *x, *residual, *weight, *post, *gate;
  const float2* stats;
  T *dx, *dresidual, *dgate;
  float *weight_lines, *branch_lines;
  uint32_t rows, period;
  int columns, walkers;
  bool pairs;
  int64_t ldgy, ldgs, ldx, ldr, ldgate, ldo;
  float inv_cols, offset, scale, residual_scale;
  int act;
};

template <typename T, bool VEC, int TPR, bool ROW_GATE>
__global__ void __launch_bounds__(TPR, kMaxWalk / TPR)
gated_backward_kernel(const BackwardArgs<T> a, int slots, uint32_t slot_bytes, uint32_t probes) {
  using PW = Pairs<T, VEC>;
  constexpr int N = PW::N, P = PW::P, ITEMS = kColumns / N;
  const int cols = a.columns, words = (cols + N - 1) / N;
  const RowShape shape = {cols, a.pairs};
  extern __shared__ __align__(128) unsigned char memory[];
  __shared__ uint64_t barriers[kMaxSlots];
  __shared__ uint32_t flags[2];
  __shared__ float sums_store[2][4][16];
  pdl_prologue();
  const int lane_in_row = threadIdx.x, walker = blockIdx.x;
  const uint32_t first = range_start(a.rows, a.walkers, walker), last = range_start(a.rows, a.walkers, walker + 1);
  Ring<T, VEC, TPR> ring;
  const bool has_gs = a.gs != nullptr;
  ring.start(barriers, memory, flags, slots, static_cast<uint32_t>(cols) * sizeof(T), slot_bytes, first, last, 3 + (ROW_GATE ? 1 : 0) + (has_gs ? 1 : 0),
             [&](int array, const T*& base, int64_t& ld) {
               base = array == 0 ? a.x : array == 1 ? a.residual : array == 2 ? a.gy : ROW_GATE && array == 3 ? a.gate : a.gs;
               ld = array == 0 ? a.ldx : array == 1 ? a.ldr : array == 2 ? a.ldgy : ROW_GATE && array == 3 ? a.ldgate : a.ldgs;
             });
  bool ok[ITEMS];
  Float2x factor[ITEMS][P], weight[ITEMS][P], sum_w[ITEMS][P], sum_k[ITEMS][P];
  const Float2x offset2 = both(a.offset);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int w = lane_in_row + i * TPR;
    ok[i] = w < words;
#pragma unroll
    for (int j = 0; j < P; ++j) weight[i][j] = sum_w[i][j] = sum_k[i][j] = both(0.f);
    if (ok[i]) {
      PW::load_shared_by_rows(a.weight, w, shape, weight[i]);
#pragma unroll
      for (int j = 0; j < P; ++j) weight[i][j] = add_f2(weight[i][j], offset2);
    }
  }
  // f of this thread's columns; without the gate where every row has its own
  auto load_factor = [&](uint32_t gate_row) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int w = lane_in_row + i * TPR;
#pragma unroll
      for (int j = 0; j < P; ++j) factor[i][j] = both(a.scale);
      if (!ok[i]) continue;
      Float2x v[P];
      if (a.post != nullptr) {
        PW::load_shared_by_rows(a.post, w, shape, v);
#pragma unroll
        for (int j = 0; j < P; ++j) factor[i][j] = mul_f2(factor[i][j], add_f2(v[j], offset2));
      }
      if (!ROW_GATE && a.gate != nullptr) {
        PW::load_shared_by_rows(a.gate + static_cast<int64_t>(gate_row) * a.ldgate, w, shape, v);
#pragma unroll
        for (int j = 0; j < P; ++j) factor[i][j] = mul_f2(factor[i][j], activate2<T>(v[j], a.act));
      }
    }
  };
  auto write_line = [&](float* line, const Float2x (&sums)[ITEMS][P]) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (!ok[i]) continue;
      const int64_t c = static_cast<int64_t>(lane_in_row + i * TPR) * N;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        float lo, hi;
        unpack_f2(sums[i][j], lo, hi);
        line[c + 2 * j] = lo;
        if (c + 2 * j + 1 < cols) line[c + 2 * j + 1] = hi;
      }
    }
  };
  uint32_t gate_row = 0, gate_end = a.rows;  // rows below gate_end share gate_row
  if (!ROW_GATE && a.gate != nullptr && first < last) {
    gate_row = first / a.period;
    gate_end = (gate_row + 1) * a.period;
  }
  load_factor(gate_row);
  const Float2x residual_scale2 = both(a.residual_scale), scale2 = both(a.scale);
  const RowAct row_act = make_row_act(a.act);
  const bool tight = slots < 2 * ring.count;  // the next row's copies need slots of this one: a barrier of their own at its end
  float2 stat = first < last ? a.stats[first] : make_float2(0.f, 0.f);  // of the next row: its latency is that of a row
  int parity = 0;
  for (uint32_t row = first; row < last; ++row, parity ^= 1) {
    if (!ROW_GATE && row >= gate_end) {
      write_line(a.branch_lines + static_cast<int64_t>(walker + gate_row) * cols, sum_k);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < P; ++j) sum_k[i][j] = both(0.f);
      ++gate_row;
      gate_end += a.period;
      load_factor(gate_row);
    }
    float r1 = stat.x, r2 = stat.y;
    if (row + 1 < last) stat = a.stats[row + 1];
    const bool landed = ring.wait(row - first, probes, TPR == 32 || tight);
    if (!landed && ring.unsound()) r1 = r2 = NAN;
    const RowView xv = ring.view(a.x, a.ldx, row, landed), rv = ring.view(a.residual, a.ldr, row, landed), gyv = ring.view(a.gy, a.ldgy, row, landed);
    const RowView gv = ROW_GATE ? ring.view(a.gate, a.ldgate, row, landed) : gyv, gsv = has_gs ? ring.view(a.gs, a.ldgs, row, landed) : gyv;
    const Float2x r12 = both(r1), r22 = both(r2);
    Float2x value[ROW_GATE ? ITEMS : 1][P];  // of the row's own gate
    Float2x acc[4] = {both(0.f), both(0.f), both(0.f), both(0.f)};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (!ok[i]) continue;
      const int w = lane_in_row + i * TPR;
      Float2x x[P], res[P], gy[P], gs[P];
      PW::load(xv, w, shape, x);
      PW::load(rv, w, shape, res);
      PW::load(gyv, w, shape, gy);
      if constexpr (ROW_GATE) {
        PW::load(gv, w, shape, value[i]);
        activate_row(value[i], row_act);
      }
#pragma unroll
      for (int j = 0; j < P; ++j) gs[j] = both(0.f);
      if (has_gs) PW::load(gsv, w, shape, gs);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        Float2x f = factor[i][j];
        if constexpr (ROW_GATE) f = mul_f2(f, value[i][j]);
        const Float2x u = mul_f2(f, mul_f2(r12, x[j]));
        const Float2x s = fma_f2(residual_scale2, res[j], u);
        const Float2x gw = mul_f2(gy[j], weight[i][j]);
        acc[0] = fma_f2(gw, s, acc[0]);
        acc[1] = fma_f2(u, gs[j], acc[1]);
        acc[2] = fma_f2(u, gw, acc[2]);
        acc[3] = fma_f2(u, s, acc[3]);
      }
    }
    float sums[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) sums[n] = pair_total(acc[n]);
    row_sums<TPR>(sums, sums_store[parity]);
    // every thread of the walker is past the row before: its slots can be filled again
    if (TPR > 32 && !tight) ring.release(row - first, row - first);
    const float c2 = r2 * r2 * r2 * (sums[0] * a.inv_cols);
    // sums 1 to 3 hold r1 f x, and grad_x takes r1 x: c1 = r1^2 (r1 <f ds, x>) / cols, c1 x = (c1 / r1) r1 x
    const float inner = sums[1] + r2 * sums[2] - c2 * sums[3];
    const Float2x minus_c2 = both(-c2), minus_c1 = both(a.post == nullptr ? 0.f : -r1 * (inner * a.inv_cols));
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (!ok[i]) continue;
      const int w = lane_in_row + i * TPR;
      const int64_t at = row * a.ldo;
      Float2x x[P], res[P], gy[P], gs[P], g[P];
      PW::load(xv, w, shape, x);
      PW::load(rv, w, shape, res);
      PW::load(gyv, w, shape, gy);
#pragma unroll
      for (int j = 0; j < P; ++j) gs[j] = both(0.f);
      if (has_gs) PW::load(gsv, w, shape, gs);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        Float2x f = factor[i][j];
        if constexpr (ROW_GATE) f = mul_f2(f, value[i][j]);
        const Float2x xr = mul_f2(r12, x[j]), gr = mul_f2(r22, gy[j]);
        const Float2x s = fma_f2(residual_scale2, res[j], mul_f2(f, xr));
        const Float2x ds = fma_f2(minus_c2, s, fma_f2(gr, weight[i][j], gs[j]));
        sum_w[i][j] = fma_f2(gr, s, sum_w[i][j]);
        if constexpr (ROW_GATE) {
          const Float2x k = mul_f2(ds, xr);
          sum_k[i][j] = fma_f2(mul_f2(scale2, value[i][j]), k, sum_k[i][j]);
          float lo, hi;
          unpack_f2(value[i][j], lo, hi);
          g[j] = mul_f2(mul_f2(factor[i][j], pack_f2(row_slope(lo, row_act), row_slope(hi, row_act))), k);
        } else {
          sum_k[i][j] = fma_f2(ds, xr, sum_k[i][j]);
        }
        x[j] = fma_f2(f, mul_f2(r12, ds), mul_f2(minus_c1, xr));
        res[j] = mul_f2(residual_scale2, ds);
      }
      PW::store(a.dx + at, w, shape, x);
      PW::store(a.dresidual + at, w, shape, res);
      if constexpr (ROW_GATE) PW::store(a.dgate + at, w, shape, g);
    }
    if (TPR == 32 || tight) {
      __syncthreads();
      ring.release(row - first, row - first + 1);
    }
  }
  ring.finish();
  write_line(a.weight_lines + static_cast<int64_t>(walker) * cols, sum_w);
  if (a.branch_lines != nullptr) write_line(a.branch_lines + static_cast<int64_t>(walker + gate_row) * cols, sum_k);
}

// Any width: one CTA per walker, the row read twice, the sums of a walker's columns kept in its lines in scratch.
template <typename T>
__global__ void __launch_bounds__(kBackwardThreads)
gated_backward_wide_kernel(const BackwardArgs<T> a, int64_t cols, bool row_gate) {
  pdl_prologue();
  __shared__ float slots[2][4][16];
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
  clear_k();
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
      const float s = stream_value(x, Num<T>::up(rr[c]), f, r1, a.residual_scale);
      const float gw = Num<T>::up(gyr[c]) * (Num<T>::up(a.weight[c]) + a.offset), u = f * x;
      sums[0] = fmaf(gw, s, sums[0]);
      if (gsr != nullptr) sums[1] = fmaf(u, Num<T>::up(gsr[c]), sums[1]);
      sums[2] = fmaf(u, gw, sums[2]);
      sums[3] = fmaf(u, s, sums[3]);
    }
    row_sums<kBackwardThreads>(sums, slots[parity]);
    const float c2 = r2 * r2 * r2 * (sums[0] * a.inv_cols);
    const float inner = sums[1] + r2 * sums[2] - c2 * sums[3];
    const float c1 = a.post == nullptr ? 0.f : r1 * r1 * r1 * (inner * a.inv_cols);
    for (int64_t c = threadIdx.x; c < cols; c += kBackwardThreads) {
      const float p = a.post == nullptr ? 1.f : Num<T>::up(a.post[c]) + a.offset;
      const float value = gr == nullptr ? 1.f : activate<T>(Num<T>::up(gr[c]), a.act);
      const float branch = a.scale * value, f = branch * p, x = Num<T>::up(xr[c]), gy = Num<T>::up(gyr[c]);
      const float s = stream_value(x, Num<T>::up(rr[c]), f, r1, a.residual_scale);
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
// a gate that rows share.  A CTA owns 32 columns; its 32 warps take every 32nd line (or gate row) each, so that all of a
// warp's loads are in flight at once, then the 32 sums are added in warp order.
constexpr int kColumnWarps = 32;
template <typename T>
struct ColumnArgs {
  const float *weight_lines, *branch_lines;
  const T *post, *gate;
  T *dweight, *dpost, *dgate;
  int64_t cols, ldgate;
  uint32_t rows, period;
  int walkers, gate_rows;  // gate_rows: 0 unless rows share gate rows
  float offset, scale, line_scale;  // line_scale: what a sum over branch_lines lacks of grad_post_weight
  int act;
};
template <typename T>
__global__ void __launch_bounds__(32 * kColumnWarps)
gated_columns_kernel(const ColumnArgs<T> a) {
  pdl_prologue();
  __shared__ float part[2][kColumnWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sum_w = 0.f, sum_p = 0.f;
  if (c < a.cols) {
    const bool branch = a.branch_lines != nullptr && a.gate_rows <= 1;
    constexpr int BATCH = 8;  // loads of either kind in flight
    for (int l0 = warp; l0 < a.walkers; l0 += BATCH * kColumnWarps) {
      float w[BATCH], p[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int l = l0 + k * kColumnWarps;
        w[k] = l < a.walkers ? a.weight_lines[l * a.cols + c] : 0.f;
        p[k] = branch && l < a.walkers ? a.branch_lines[l * a.cols + c] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        sum_w += w[k];
        sum_p += p[k];
      }
    }
    if (a.branch_lines != nullptr && a.gate_rows > 1) {
      const float p = a.post == nullptr ? 1.f : Num<T>::up(a.post[c]) + a.offset;
      for (int g = warp; g < a.gate_rows; g += kColumnWarps) {
        // walkers whose rows meet this gate row's: those from the one that holds its first row to the one that holds its last
        const uint64_t lo = static_cast<uint64_t>(g) * a.period, hi = lo + a.period;
        int w = a.rows == 0 ? 0 : static_cast<int>(lo * a.walkers / a.rows);
        while (w > 0 && range_start(a.rows, a.walkers, w) > lo) --w;
        while (w + 1 < a.walkers && range_start(a.rows, a.walkers, w + 1) <= lo) ++w;
        float k = 0.f;
        for (; w < a.walkers && range_start(a.rows, a.walkers, w) < hi; ++w)
          if (range_start(a.rows, a.walkers, w + 1) > range_start(a.rows, a.walkers, w)) k += a.branch_lines[static_cast<int64_t>(w + g) * a.cols + c];
        const float value = activate<T>(Num<T>::up(a.gate[g * a.ldgate + c]), a.act);
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
    for (int k = 0; k < kColumnWarps; ++k) {
      sum_w += part[0][k][lane];
      sum_p += part[1][k][lane];
    }
    a.dweight[c] = Num<T>::down(sum_w);
    if (a.gate_rows == 1) {
      const float value = activate<T>(Num<T>::up(a.gate[c]), a.act), p = a.post == nullptr ? 1.f : Num<T>::up(a.post[c]) + a.offset;
      a.dgate[c] = Num<T>::down(a.scale * p * activation_slope(value, a.act) * sum_p);
      sum_p *= a.scale * value;
    }
    if (a.dpost != nullptr) a.dpost[c] = Num<T>::down(a.line_scale * sum_p);
  }
}

// Rows of up to kWalkColumns columns go through a ring, wider ones through the CTAs of gated_backward_wide_kernel.
struct BackwardPlan {
  bool walk;
  WalkPlan w;
  int64_t weight_lines, branch_lines;
};
BackwardPlan plan_backward(int64_t rows, int64_t cols, int64_t gate_rows, size_t element) {
  BackwardPlan p;
  p.walk = cols <= kWalkColumns;
  const bool by_group = gate_rows > 1 && gate_rows < rows;
  if (p.walk) {
    p.w = plan_walk(rows, cols, element);
  } else {
    p.w.walkers = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rows, static_cast<int64_t>(sm_count()) * 2)));
  }
  p.weight_lines = p.w.walkers;
  p.branch_lines = p.w.walkers + (by_group ? gate_rows : 0);
  return p;
}

// B200_GATED_WAIT_PROBES=<n> in the environment replaces the limit of a wait for a row's copies (read at every call; with 0 every
// row is fetched with ordinary loads).
uint32_t wait_probes() {
  const char* v = std::getenv("B200_GATED_WAIT_PROBES");
  return v != nullptr ? static_cast<uint32_t>(std::strtoul(v, nullptr, 10)) : kSpinLimit;
}

template <typename T, bool VEC, int TPR, bool ROW_GATE>
int launch_backward(const BackwardArgs<T>& a, const WalkPlan& p, cudaStream_t st) {
  constexpr auto kernel = gated_backward_kernel<T, VEC, TPR, ROW_GATE>;
  if (int rc = allow_smem<kernel, kRingBytes>("gated_backward_kernel")) return rc;
  launch(kernel, static_cast<unsigned>(p.walkers), TPR, static_cast<size_t>(p.slots) * p.slot_bytes, st, a, p.slots, p.slot_bytes, wait_probes());
  return after_launch("gated_backward_kernel");
}

template <typename T, bool VEC>
int run_walk_back(const BackwardArgs<T>& a, const WalkPlan& p, bool row_gate, cudaStream_t st) {
#define B200_WALK(TPR) return row_gate ? launch_backward<T, VEC, TPR, true>(a, p, st) : launch_backward<T, VEC, TPR, false>(a, p, st)
  switch (p.tpr) {
    case 32: B200_WALK(32);
    case 64: B200_WALK(64);
    case 128: B200_WALK(128);
    case 256: B200_WALK(256);
    default: B200_WALK(512);
  }
#undef B200_WALK
}

template <typename T>
int run_backward(BackwardArgs<T> a, ColumnArgs<T> c, int64_t cols, const BackwardPlan& p, bool vec, bool row_gate, cudaStream_t st) {
  int rc;
  if (!p.walk) {
    launch(gated_backward_wide_kernel<T>, static_cast<unsigned>(a.walkers), kBackwardThreads, 0, st, a, cols, row_gate);
    rc = after_launch("gated_backward_wide_kernel");
  } else {
    rc = vec ? run_walk_back<T, true>(a, p.w, row_gate, st) : run_walk_back<T, false>(a, p.w, row_gate, st);
  }
  if (rc) return rc;
  launch(gated_columns_kernel<T>, static_cast<unsigned>(ceil_div(cols, 32)), 32 * kColumnWarps, 0, st, c);
  return after_launch("gated_columns_kernel");
}

}  // namespace

unsigned int gated_backward_wait_timeouts() { return read_wait_timeouts(); }

}  // namespace b200

using namespace b200;

extern "C" int b200_gated_add_rms_norm_backward_scratch_bytes(int64_t rows, int64_t cols, int64_t gate_rows, int dtype, size_t* bytes) {
  B200_REQUIRE_PTR(bytes);
  if (int rc = check_shapes(__func__, rows, cols, gate_rows, nullptr, dtype, kIdentity)) return rc;
  if (int rc = check_device()) return rc;
  const BackwardPlan p = plan_backward(rows, cols, gate_rows, dtype_size(dtype));
  *bytes = static_cast<size_t>(p.weight_lines + p.branch_lines) * static_cast<size_t>(cols) * sizeof(float);
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
  for (const void* p : all)
    if (!aligned(p, es)) return fail(B200_ERR_ALIGNMENT, "%s: pointer not aligned to the element size", __func__);
  if (!aligned(stats, 8)) return fail(B200_ERR_ALIGNMENT, "%s: stats must be 8-byte aligned", __func__);
  if (int rc = check_device()) return rc;
  if (rows == 0) {
    if (cudaMemsetAsync(grad_weight, 0, cols * es, static_cast<cudaStream_t>(stream)) != cudaSuccess ||
        (grad_post_weight && cudaMemsetAsync(grad_post_weight, 0, cols * es, static_cast<cudaStream_t>(stream)) != cudaSuccess) ||
        (grad_gate && cudaMemsetAsync(grad_gate, 0, gate_rows * cols * es, static_cast<cudaStream_t>(stream)) != cudaSuccess))
      return fail(B200_ERR_LAUNCH, "%s: %s", __func__, cudaGetErrorString(cudaGetLastError()));
    return B200_OK;
  }
  const Access access = access_of(es, cols, {grad_y, grad_s, x, residual, weight, post_weight, gate, grad_x, grad_residual, grad_gate},
                                  {ldgy, grad_s == nullptr ? 0 : ldgs, ldx, ldr, gate != nullptr && gate_rows > 1 ? ldgate : 0});
  const BackwardPlan p = plan_backward(rows, cols, gate == nullptr ? 0 : gate_rows, es);
  const size_t need = static_cast<size_t>(p.weight_lines + p.branch_lines) * static_cast<size_t>(cols) * sizeof(float);
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
    a.branch_lines = post_weight == nullptr && !shared_gate ? nullptr : a.weight_lines + p.weight_lines * cols;
    a.rows = static_cast<uint32_t>(rows), a.period = shared_gate ? static_cast<uint32_t>(rows / gate_rows) : 1;
    a.columns = static_cast<int>(cols), a.walkers = p.w.walkers, a.pairs = access == kPairs;
    a.ldgy = ldgy, a.ldgs = ldgs, a.ldx = ldx, a.ldr = ldr, a.ldgate = ldgate, a.ldo = cols;
    a.inv_cols = 1.f / static_cast<float>(cols), a.offset = static_cast<float>(offset), a.scale = static_cast<float>(scale);
    a.residual_scale = static_cast<float>(residual_scale), a.act = activation;
    ColumnArgs<T> c;
    c.weight_lines = a.weight_lines, c.branch_lines = a.branch_lines, c.post = a.post, c.gate = a.gate;
    c.dweight = static_cast<T*>(grad_weight), c.dpost = static_cast<T*>(grad_post_weight), c.dgate = a.dgate;
    c.cols = cols, c.ldgate = ldgate, c.rows = a.rows, c.period = a.period;
    c.walkers = p.w.walkers, c.gate_rows = shared_gate ? static_cast<int>(gate_rows) : 0;
    c.offset = a.offset, c.scale = a.scale, c.line_scale = gate == nullptr ? a.scale : 1.f, c.act = activation;
    return run_backward<T>(a, c, cols, p, access == kWords, row_gate, static_cast<cudaStream_t>(stream));
  });
  return B200_OK;
}
