// Token embedding: out[t] = scale * weight[ids[t]], and the gradient of the table.
//
// Forward: one warp copies up to 128 words of a row; bound by HBM (the ids, the rows read and written).
//
// Backward: grad_weight[v] = scale * sum over t with ids[t] = v of grad_out[t], ascending t, fp32, one rounding.
// Bound by HBM: grad_out read once, every row of the table written once.  Three launches:
//   1. order: CTA c owns a range of at most 1024 rows of the table.  It goes over all ids, counts those below its range
//      (that is where its part of the sorted list starts) and those of each of its rows, and lists its tokens by (id, t).
//      No CTA waits for another.  Rows that no token has are zeroed here.
//   2. sums: the sorted list is cut into units of equal length, so that a frequent token is spread over many CTAs.  A run
//      of equal ids inside a unit goes straight to its row; the parts of one that crosses units go to scratch in fp32.
//   3. join: adds up the parts of such runs, in order.
// No pointer is __restrict__: the second and third kernel begin with loads of what the kernel before them wrote (see ld_kept).
// No atomics on values and a fixed order of every sum: the same inputs give the same bits.
#include <algorithm>

#include "common.cuh"

namespace b200 {
namespace {

constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;
constexpr int kMaxRange = 1024;   // rows of the table per CTA of the order kernel
constexpr int kSumThreads = 128;  // one load of each row per thread: a tile of columns
constexpr int kMaxUnit = 32;      // sorted tokens per unit

template <typename T, bool VEC>
struct Word;
template <typename T>
struct Word<T, true> {
  static constexpr int N = Num<T>::kVec;
  using Raw = uint4;
  static __device__ __forceinline__ Raw load(const T* p) { return ld_stream(p); }
  static __device__ __forceinline__ Raw load_table(const T* p) { return ld_kept(p); }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[N]) { Num<T>::unpack(r, f); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[N]) { st_stream(p, Num<T>::pack(f)); }
};
template <typename T>
struct Word<T, false> {
  static constexpr int N = 1;
  using Raw = T;
  static __device__ __forceinline__ Raw load(const T* p) { return *p; }
  static __device__ __forceinline__ Raw load_table(const T* p) { return *p; }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[1]) { f[0] = Num<T>::up(r); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[1]) { *p = Num<T>::down(f[0]); }
};

// ids are int32 or int64; one outside [0, vocab) has no row
template <typename I>
__device__ __forceinline__ int row_of(I id, int64_t vocab) {
  return id >= 0 && static_cast<int64_t>(id) < vocab ? static_cast<int>(id) : -1;
}

template <typename T, typename I, bool VEC>
__global__ void __launch_bounds__(256)
embedding_kernel(const I* ids, const T* weight, T* out, int64_t tokens, int64_t vocab, int64_t words,
                 int64_t ldw, int64_t ldo, float scale) {
  using W = Word<T, VEC>;
  constexpr int N = W::N, ITEMS = 4;
  pdl_prologue();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32;
  if (t >= tokens) return;
  const int row = row_of(ids[t], vocab);
  const int64_t w0 = static_cast<int64_t>(blockIdx.y) * (32 * ITEMS) + threadIdx.x % 32;
  typename W::Raw v[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (row >= 0 && w0 + i * 32 < words) v[i] = W::load_table(weight + row * ldw + (w0 + i * 32) * N);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (w0 + i * 32 >= words) continue;
    float f[N];
    if (row >= 0) W::unpack(v[i], f);
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = row >= 0 ? f[j] * scale : 0.f;
    W::store(out + t * ldo + (w0 + i * 32) * N, f);
  }
}

// The tokens by (id, t): token[i] and id[i] for i < *count.
template <typename T, typename I>
__global__ void __launch_bounds__(kOrderThreads)
embedding_order_kernel(const I* ids, int tokens, int64_t vocab, int padding, int range, int32_t* token,
                       int32_t* id, int32_t* count, T* grad_weight, int64_t cols) {
  constexpr int AHEAD = 8;
  extern __shared__ int place[];  // [warp][row of the range]: first the warp's tokens of the row, then where they go
  __shared__ int totals[kMaxRange];
  __shared__ int fold[kOrderWarps];
  __shared__ int next_row;
  pdl_prologue();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t first_row = static_cast<int64_t>(blockIdx.x) * range;
  const int rows = static_cast<int>(min(static_cast<int64_t>(range), vocab - first_row));
  if (threadIdx.x == 0) next_row = 0;
  for (int i = threadIdx.x; i < kOrderWarps * range; i += kOrderThreads) place[i] = 0;
  __syncthreads();
  // the ids in one contiguous piece per warp, so that piece order is token order
  const int piece = (tokens + kOrderWarps - 1) / kOrderWarps;
  auto piece_start = [&](int p) { return static_cast<int>(min(static_cast<int64_t>(tokens), static_cast<int64_t>(p) * piece)); };
  const int begin = piece_start(warp), end = piece_start(warp + 1);
  int below = 0;
  // the rows of eight batches of a warp's tokens at a time; -1: none, also for padding
  int row[AHEAD];
  auto fetch = [&](int t0, int stop) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int t = t0 + k * 32 + lane;
      row[k] = t < stop ? row_of(ids[t], vocab) : -1;
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (row[k] == padding) row[k] = -1;
  };
  for (int t0 = begin; t0 < end; t0 += 32 * AHEAD) {
    fetch(t0, end);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int64_t at = row[k] - first_row;
      if (row[k] >= 0 && at < 0) ++below;
      if (at >= 0 && at < rows) atomicAdd(&place[warp * range + at], 1);
    }
  }
  below = __reduce_add_sync(0xffffffffu, below);
  if (lane == 0) fold[warp] = below;
  __syncthreads();
  int start = 0;
#pragma unroll
  for (int w = 0; w < kOrderWarps; ++w) start += fold[w];
  // exclusive sums: over the warps of a row, then over the rows
  int mine = 0;
  if (threadIdx.x < rows) {
#pragma unroll 8
    for (int w = 0; w < kOrderWarps; ++w) {
      const int n = place[w * range + threadIdx.x];
      place[w * range + threadIdx.x] = mine;
      mine += n;
    }
    totals[threadIdx.x] = mine;
  }
  int scan = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += v;
  }
  __syncthreads();  // `fold` has been read
  if (lane == 31) fold[warp] = scan;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kOrderWarps; ++w) {
    if (w < warp) before += fold[w];
    all += fold[w];
  }
  if (threadIdx.x < rows) {
    const int at = start + before + scan - mine;
#pragma unroll 8
    for (int w = 0; w < kOrderWarps; ++w) place[w * range + threadIdx.x] += at;
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *count = start + all;
  __syncthreads();
  // half of the warps list the tokens, two pieces each; the others begin with the rows without tokens, whose stores then hide
  // the latency of the first half's loads
  for (int p = warp; warp < kOrderWarps / 2 && p < kOrderWarps; p += kOrderWarps / 2) {
    const int stop = piece_start(p + 1);
    int* next = place + p * range;
    for (int t0 = piece_start(p); t0 < stop; t0 += 32 * AHEAD) {
      fetch(t0, stop);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int64_t at = row[k] - first_row;
        const bool here = at >= 0 && at < rows;
        const unsigned active = __ballot_sync(0xffffffffu, here);
        if (active == 0) continue;
        if (here) {
          const unsigned same = __match_any_sync(active, row[k]);
          const int rank = __popc(same & ((1u << lane) - 1));
          const int to = next[at] + rank;
          __syncwarp(active);
          if (rank == 0) next[at] += __popc(same);
          token[to] = t0 + k * 32 + lane;
          id[to] = row[k];
        }
        __syncwarp();
      }
    }
  }
  // rows without tokens: words between the 16-byte boundaries, single elements around them
  constexpr int64_t V = Num<T>::kVec;
  for (;;) {
    int r = 0;
    if (lane == 0) r = atomicAdd(&next_row, 1);  // whichever warp takes it writes the same zeros
    r = __shfl_sync(0xffffffffu, r, 0);
    if (r >= rows) break;
    if (totals[r] != 0) continue;
    T* out = grad_weight + (first_row + r) * cols;
    const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(out) / sizeof(T) % V);
    const int64_t head = min(cols, (V - off) % V), words = (cols - head) / V, tail = head + words * V;
    if (lane < head) out[lane] = Num<T>::down(0.f);
    for (int64_t w = lane; w < words; w += 32) st_stream(out + head + w * V, make_uint4(0, 0, 0, 0));
    if (tail + lane < cols) out[tail + lane] = Num<T>::down(0.f);
  }
}

template <int N>
__device__ __forceinline__ void put_part(float* p, const float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) p[j] = v[j];
}

// parts: [unit][0: the run that came from the unit before, 1: the run that goes on in the next unit and began in this one][cols]
template <typename T, bool VEC>
__global__ void __launch_bounds__(kSumThreads)
embedding_sum_kernel(const T* grad, const int32_t* token, const int32_t* id, const int32_t* count,
                     T* grad_weight, float* parts, int unit, int capacity, int64_t words, int64_t cols, int64_t ldg, float scale) {
  using W = Word<T, VEC>;
  constexpr int N = W::N, AHEAD = 8;
  __shared__ int tokens[kMaxUnit], ids[kMaxUnit + 2];
  pdl_prologue();
  // all three loads at once: what lies behind the list's end is read and not used
  const int first = blockIdx.x * unit, i = first + static_cast<int>(threadIdx.x);
  const int mine = threadIdx.x < unit && i < capacity ? token[i] : 0;
  const int my_id = threadIdx.x < unit + 2 && i >= 1 && i <= capacity ? id[i - 1] : -1;
  const int total = *count;
  if (first >= total) return;
  const int n = min(unit, total - first);
  if (threadIdx.x < n) tokens[threadIdx.x] = mine;
  if (threadIdx.x < n + 2) ids[threadIdx.x] = i <= total ? my_id : -1;  // with the neighbours of the unit
  __syncthreads();
  const int64_t w = static_cast<int64_t>(blockIdx.y) * kSumThreads + threadIdx.x;
  if (w >= words) return;
  const T* from = grad + w * N;
  float* part = parts + static_cast<int64_t>(blockIdx.x) * 2 * cols + w * N;
  float sum[N];
#pragma unroll
  for (int j = 0; j < N; ++j) sum[j] = 0.f;
  bool carried = ids[0] == ids[1];  // the run began in an earlier unit
  for (int i0 = 0; i0 < n; i0 += AHEAD) {
    typename W::Raw v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i0 + k < n) v[k] = W::load(from + tokens[i0 + k] * ldg);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (i0 + k >= n) break;
      float f[N];
      W::unpack(v[k], f);
#pragma unroll
      for (int j = 0; j < N; ++j) sum[j] += f[j];
      const int here = ids[i0 + k + 1];
      const bool goes_on = here == ids[i0 + k + 2];
      if (goes_on && i0 + k + 1 < n) continue;
      if (carried) {
        put_part(part, sum);
      } else if (goes_on) {
        put_part(part + cols, sum);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] *= scale;
        W::store(grad_weight + here * cols + w * N, sum);
      }
      carried = false;
#pragma unroll
      for (int j = 0; j < N; ++j) sum[j] = 0.f;
    }
  }
}

// Adds up the parts of the runs that cross units.  A CTA looks after kJoinUnits units and 128 columns.  Each warp takes some
// of the runs that begin in these units and go on; one of more than kLongRun parts is added up by all warps, each an equal
// share of its parts, the shares in warp order.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kJoinColumns = 128;
constexpr int kJoinUnits = 32, kLongRun = 64;

// the last unit that the run of unit `begin` reaches: 32 units probed at a time, next to it first
__device__ __forceinline__ int last_unit(const int32_t* id, int run, int begin, int units, int unit) {
  const int lane = threadIdx.x & 31;
  int low = begin + 1, high = units - 1, step = 1;
  while (low < high) {
    const int64_t probe = low + static_cast<int64_t>(lane + 1) * step;
    const int reached = __popc(__ballot_sync(0xffffffffu, probe <= high && id[min(probe, static_cast<int64_t>(high)) * unit] == run));
    low += reached * step;
    if (reached < 32) high = min(high, low + step - 1);
    step = max(1, (high - low + 31) / 32);
  }
  return low;
}

__device__ __forceinline__ float4 add_parts(const float* parts, int begin, int from, int to, int64_t cols, int64_t c) {
  const bool words = cols % 4 == 0;  // of four columns
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = from; i < to; ++i) {
    const float* part = parts + (static_cast<int64_t>(begin + i) * 2 + (i == 0 ? 1 : 0)) * cols + c;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (words && c < cols) {
      v = *reinterpret_cast<const float4*>(part);
    } else {
      if (c < cols) v.x = part[0];
      if (c + 1 < cols) v.y = part[1];
      if (c + 2 < cols) v.z = part[2];
      if (c + 3 < cols) v.w = part[3];
    }
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  return sum;
}

template <typename T>
__global__ void __launch_bounds__(kJoinThreads)
embedding_join_kernel(const int32_t* id, const int32_t* count, const float* parts, T* grad_weight, int unit, int64_t cols, float scale) {
  __shared__ int long_begin[kJoinUnits], long_parts[kJoinUnits];
  __shared__ int found;
  __shared__ float4 share[kJoinWarps][32];
  if (threadIdx.x == 0) found = 0;
  pdl_prologue();
  const int total = *count, units = (total + unit - 1) / unit;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int u0 = blockIdx.x * kJoinUnits;
  if (u0 + 1 >= units) return;
  const int64_t c = static_cast<int64_t>(blockIdx.y) * kJoinColumns + lane * 4;
  bool begins = false;  // a run begins in this lane's unit and goes on in the next
  int my_run = 0;
  if (u0 + lane + 1 < units) {
    const int64_t first = static_cast<int64_t>(u0 + lane) * unit;
    my_run = id[first + unit - 1];
    const int behind = id[first + unit], start = id[first], before = first == 0 ? -1 : id[first - 1];
    begins = behind == my_run && (start != my_run || before != my_run);
  }
  __syncthreads();  // `found` is zero
  unsigned todo = __ballot_sync(0xffffffffu, begins);
  for (int k = 0; todo != 0; ++k, todo &= todo - 1) {
    if (k % kJoinWarps != warp) continue;
    const int at = __ffs(todo) - 1, begin = u0 + at, run = __shfl_sync(0xffffffffu, my_run, at);
    const int n = last_unit(id, run, begin, units, unit) - begin + 1;  // parts: the second of unit `begin`, the first of the others
    if (n > kLongRun) {
      if (lane == 0) {
        const int slot = atomicAdd(&found, 1);  // in any order: the runs do not meet
        long_begin[slot] = begin;
        long_parts[slot] = n;
      }
      continue;
    }
    const float4 sum = add_parts(parts, begin, 0, n, cols, c);
    T* out = grad_weight + run * cols + c;
    if (c < cols) out[0] = Num<T>::down(sum.x * scale);
    if (c + 1 < cols) out[1] = Num<T>::down(sum.y * scale);
    if (c + 2 < cols) out[2] = Num<T>::down(sum.z * scale);
    if (c + 3 < cols) out[3] = Num<T>::down(sum.w * scale);
  }
  __syncthreads();
  const int runs = found;
  for (int k = 0; k < runs; ++k) {
    const int begin = long_begin[k], n = long_parts[k], run = id[static_cast<int64_t>(begin) * unit + unit - 1];
    const float4 sum = add_parts(parts, begin, static_cast<int>(static_cast<int64_t>(n) * warp / kJoinWarps), static_cast<int>(static_cast<int64_t>(n) * (warp + 1) / kJoinWarps), cols, c);
    __syncthreads();  // the run before has been read
    share[warp][lane] = sum;
    __syncthreads();
    const int64_t column = static_cast<int64_t>(blockIdx.y) * kJoinColumns + threadIdx.x;
    if (threadIdx.x < kJoinColumns && column < cols) {
      float all = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) all += reinterpret_cast<const float*>(share[w])[threadIdx.x];
      grad_weight[run * cols + column] = Num<T>::down(all * scale);
    }
  }
}

struct Scratch {
  int32_t *token, *id, *count;
  float* parts;
};
int unit_length(int64_t tokens) { return tokens >= 8192 ? kMaxUnit : 8; }
size_t scratch_layout(int64_t tokens, int64_t cols, char* base, Scratch* out) {
  const int64_t units = ceil_div(tokens, unit_length(tokens));
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 15) / 16 * 16;
    return base + here;
  };
  Scratch s;
  s.count = reinterpret_cast<int32_t*>(take(4));
  s.token = reinterpret_cast<int32_t*>(take(static_cast<size_t>(tokens) * 4));
  s.id = reinterpret_cast<int32_t*>(take(static_cast<size_t>(tokens) * 4));
  s.parts = reinterpret_cast<float*>(take(static_cast<size_t>(units) * 2 * static_cast<size_t>(cols) * 4));
  if (out != nullptr) *out = s;
  return at;
}

int check_sizes(const char* fn, int64_t tokens, int64_t vocab, int64_t cols, int dtype) {
  if (!dtype_ok(dtype)) return fail(B200_ERR_DTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (tokens < 0 || vocab < 0 || cols < 0) return fail(B200_ERR_SHAPE, "%s: negative size", fn);
  if (tokens > (1LL << 30) || vocab > 0x7fffffffLL) return fail(B200_ERR_SHAPE, "%s: tokens=%lld exceeds 2^30 or vocab=%lld 2^31-1", fn, (long long)tokens, (long long)vocab);
  if (cols > 65535LL * 128) return fail(B200_ERR_SHAPE, "%s: cols=%lld exceeds %lld", fn, (long long)cols, 65535LL * 128);
  return B200_OK;
}

template <typename T, typename I>
int run_backward(const void* grad_out, const void* ids, void* grad_weight, int64_t tokens, int64_t vocab, int64_t cols, int64_t ldg,
                 int64_t padding, float scale, const Scratch& s, cudaStream_t st) {
  constexpr int V = Num<T>::kVec;
  const T* g = static_cast<const T*>(grad_out);
  T* out = static_cast<T*>(grad_weight);
  const bool vec = cols % V == 0 && ldg % V == 0 && aligned(g, 16) && aligned(out, 16);
  const int64_t ctas = std::max<int64_t>(sm_count(), ceil_div(vocab, kMaxRange));
  const int range = static_cast<int>(ceil_div(vocab, ctas));
  const size_t smem = static_cast<size_t>(range) * kOrderWarps * sizeof(int);
  auto order = embedding_order_kernel<T, I>;
  if (cudaFuncSetAttribute(order, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
    return fail(B200_ERR_LAUNCH, "embedding_order_kernel: %s", cudaGetErrorString(cudaGetLastError()));
  const int pad = padding >= 0 && padding < vocab ? static_cast<int>(padding) : -1;
  launch(order, static_cast<unsigned>(ceil_div(vocab, range)), kOrderThreads, smem, st, static_cast<const I*>(ids), static_cast<int>(tokens), vocab, pad,
         range, s.token, s.id, s.count, out, cols);
  if (int rc = after_launch("embedding_order_kernel")) return rc;
  if (tokens == 0) return B200_OK;
  const int unit = unit_length(tokens);
  const int64_t words = vec ? cols / V : cols, units = ceil_div(tokens, unit);
  const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(ceil_div(words, kSumThreads)));
  if (vec)
    launch(embedding_sum_kernel<T, true>, grid, kSumThreads, 0, st, g, s.token, s.id, s.count, out, s.parts, unit, static_cast<int>(tokens), words, cols, ldg, scale);
  else
    launch(embedding_sum_kernel<T, false>, grid, kSumThreads, 0, st, g, s.token, s.id, s.count, out, s.parts, unit, static_cast<int>(tokens), words, cols, ldg, scale);
  if (int rc = after_launch("embedding_sum_kernel")) return rc;
  if (units > 1) {
    const dim3 joins(static_cast<unsigned>(ceil_div(units - 1, kJoinUnits)), static_cast<unsigned>(ceil_div(cols, kJoinColumns)));
    launch(embedding_join_kernel<T>, joins, kJoinThreads, 0, st, s.id, s.count, static_cast<const float*>(s.parts), out, unit, cols, scale);
    return after_launch("embedding_join_kernel");
  }
  return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_embedding(const void* ids, const void* weight, void* out, int64_t tokens, int64_t vocab, int64_t cols, int64_t ldw,
                              int64_t ldo, int ids_64, int dtype, double scale, void* stream) {
  if (int rc = check_sizes(__func__, tokens, vocab, cols, dtype)) return rc;
  if (tokens == 0 || cols == 0) return B200_OK;
  B200_REQUIRE_PTR(ids);
  if (vocab > 0) B200_REQUIRE_PTR(weight);
  B200_REQUIRE_PTR(out);
  if (ldw < cols || ldo < cols) return fail(B200_ERR_SHAPE, "%s: leading dimension smaller than cols", __func__);
  const size_t es = dtype_size(dtype);
  if (!aligned(weight, es) || !aligned(out, es) || !aligned(ids, ids_64 ? 8 : 4)) return fail(B200_ERR_ALIGNMENT, "%s: pointer not aligned to its element size", __func__);
  if (int rc = check_device()) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  B200_DISPATCH_DTYPE(dtype, T, {
    const bool vec = cols % Num<T>::kVec == 0 && ldw % Num<T>::kVec == 0 && ldo % Num<T>::kVec == 0 && aligned(weight, 16) && aligned(out, 16);
    const int64_t words = vec ? cols / Num<T>::kVec : cols;
    const dim3 grid(static_cast<unsigned>(ceil_div(tokens, 8)), static_cast<unsigned>(ceil_div(words, 128)));
    const T* w = static_cast<const T*>(weight);
    T* o = static_cast<T*>(out);
    const float sc = static_cast<float>(scale);
    if (ids_64) {
      const int64_t* i = static_cast<const int64_t*>(ids);
      if (vec) launch(embedding_kernel<T, int64_t, true>, grid, 256, 0, st, i, w, o, tokens, vocab, words, ldw, ldo, sc);
      else launch(embedding_kernel<T, int64_t, false>, grid, 256, 0, st, i, w, o, tokens, vocab, words, ldw, ldo, sc);
    } else {
      const int32_t* i = static_cast<const int32_t*>(ids);
      if (vec) launch(embedding_kernel<T, int32_t, true>, grid, 256, 0, st, i, w, o, tokens, vocab, words, ldw, ldo, sc);
      else launch(embedding_kernel<T, int32_t, false>, grid, 256, 0, st, i, w, o, tokens, vocab, words, ldw, ldo, sc);
    }
  });
  return after_launch("embedding_kernel");
}

extern "C" int b200_embedding_backward_scratch_bytes(int64_t tokens, int64_t vocab, int64_t cols, size_t* bytes) {
  B200_REQUIRE_PTR(bytes);
  if (int rc = check_sizes(__func__, tokens, vocab, cols, B200_F32)) return rc;
  *bytes = scratch_layout(tokens, cols, nullptr, nullptr);
  return B200_OK;
}

extern "C" int b200_embedding_backward(const void* grad_out, const void* ids, void* grad_weight, int64_t tokens, int64_t vocab, int64_t cols,
                                       int64_t ldg, int64_t padding_idx, int ids_64, int dtype, double scale, void* scratch, size_t scratch_bytes,
                                       void* stream) {
  if (int rc = check_sizes(__func__, tokens, vocab, cols, dtype)) return rc;
  if (vocab == 0 || cols == 0) return B200_OK;
  B200_REQUIRE_PTR(grad_weight);
  B200_REQUIRE_PTR(scratch);
  if (tokens > 0) {
    B200_REQUIRE_PTR(grad_out);
    B200_REQUIRE_PTR(ids);
    if (ldg < cols) return fail(B200_ERR_SHAPE, "%s: leading dimension smaller than cols", __func__);
  }
  const size_t es = dtype_size(dtype);
  if (!aligned(grad_out, es) || !aligned(grad_weight, es) || !aligned(ids, ids_64 ? 8 : 4))
    return fail(B200_ERR_ALIGNMENT, "%s: pointer not aligned to its element size", __func__);
  if (int rc = check_device()) return rc;
  Scratch s;
  const size_t need = scratch_layout(tokens, cols, static_cast<char*>(scratch), &s);
  if (scratch_bytes < need || !aligned(scratch, 16))
    return fail(B200_ERR_SCRATCH, "%s: scratch needs %zu bytes, 16-byte aligned (got %zu)", __func__, need, scratch_bytes);
  const float sc = static_cast<float>(scale);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  B200_DISPATCH_DTYPE(dtype, T, {
    if (ids_64) return (run_backward<T, int64_t>(grad_out, ids, grad_weight, tokens, vocab, cols, ldg, padding_idx, sc, s, st));
    return (run_backward<T, int32_t>(grad_out, ids, grad_weight, tokens, vocab, cols, ldg, padding_idx, sc, s, st));
  });
  return B200_OK;
}
