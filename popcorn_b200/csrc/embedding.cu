// Token embedding: out[t] = scale * weight[ids[t]], and the gradient of the table.
//
// Forward: one warp copies up to 128 words of a row; bound by HBM (the ids, the rows read and written).
//
// Backward: grad_weight[v] = scale * sum over t with ids[t] = v of grad_out[t], ascending t, fp32, one rounding.
// Bound by HBM: grad_out read once, every row of the table written once.  Three launches:
//   1. order: CTA c owns a range of at most 1024 rows of the table.  It goes over all ids, counts those below its range
//      (that is where its part of the sorted list starts) and those of each of its rows, and lists its tokens by (id, t).
//      No CTA waits for another.  Meanwhile eight of its warps begin to zero the rows that no token has.
//   2. sums: the sorted list is cut into units of equal length, so that a frequent token is spread over many CTAs.  A run
//      of equal ids inside a unit goes straight to its row; the parts of one that crosses units go to scratch in fp32.
//   3. join: adds up the parts of such runs, in order, beside the zeroing of the rest of the rows that no token has.
// The zeros are most of what is written for a large table; spread over the first and third launch they hide the latency
// of the listing and of the joining (65536 tokens, fp16 [131072, 4096]: 278 us with all of them in the first, 258 with this).
// No pointer is __restrict__: the second and third kernel begin with loads of what the kernel before them wrote (see ld_kept).
// No atomics on values and a fixed order of every sum: the same inputs give the same bits.
#include <algorithm>

#include "common.cuh"
#include "tma.cuh"

namespace b200 {
namespace {

constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;
constexpr int kListWarps = kOrderWarps - 8;  // list the tokens, one piece of them each; the others zero rows meanwhile
constexpr int kMaxRange = 1024;   // rows of the table per CTA of the order kernel
constexpr int kSumThreads = 128;  // one load of each row per thread: a tile of columns
constexpr int kMaxUnit = 64;      // sorted tokens per unit

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

// Zeroing of table rows by bulk copies out of a zeroed piece of shared memory, eight threads a row and four rows a warp:
// the copy engine keeps the memory busy by itself (16-byte stores of eight warps per SM reached 3.6 TB/s).
constexpr int kZeroBytes = 1024, kZeroLanes = 8, kZeroRows = 32 / kZeroLanes;
struct Zeros {
  uint4 words[kZeroBytes / 16];
  __device__ __forceinline__ void clear(int threads) {
    for (int i = threadIdx.x; i < kZeroBytes / 16; i += threads) words[i] = make_uint4(0, 0, 0, 0);
    fence_async_smem();  // before the barrier behind which the copies are issued
  }
};
// this thread's copies of a row: what lies between 16-byte boundaries; single elements around it
template <typename T>
__device__ __forceinline__ void zero_row(const Zeros& zeros, T* out, int64_t cols) {
  const int part = threadIdx.x % kZeroLanes;
  unsigned char* begin = reinterpret_cast<unsigned char*>(out);
  unsigned char* end = reinterpret_cast<unsigned char*>(out + cols);
  unsigned char* from = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(begin) + 15) & ~static_cast<uintptr_t>(15));
  unsigned char* to = reinterpret_cast<unsigned char*>(reinterpret_cast<uintptr_t>(end) & ~static_cast<uintptr_t>(15));
  if (from >= to) from = to = end;
  for (T* p = out + part; reinterpret_cast<unsigned char*>(p) < from; p += kZeroLanes) *p = Num<T>::down(0.f);
  for (T* p = reinterpret_cast<T*>(to) + part; reinterpret_cast<unsigned char*>(p) < end; p += kZeroLanes) *p = Num<T>::down(0.f);
  if (cols * sizeof(T) % 128 != 0) {
    for (from += part * 16; from < to; from += kZeroLanes * 16) st_stream(from, make_uint4(0, 0, 0, 0));
    return;
  }
  for (from += part * kZeroBytes; from < to; from += kZeroLanes * kZeroBytes)
    bulk_store(from, zeros.words, static_cast<uint32_t>(min(static_cast<int64_t>(to - from), static_cast<int64_t>(kZeroBytes))));
}

// The tokens by (id, t): token[i] and id[i] for i < *count.
template <typename T, typename I>
__global__ void __launch_bounds__(kOrderThreads)
embedding_order_kernel(const I* ids, int tokens, int64_t vocab, int padding, int range, int32_t* token,
                       int32_t* id, int32_t* count, uint8_t* hit, int32_t* resume, T* grad_weight, int64_t cols) {
  constexpr int AHEAD = 8;
  extern __shared__ int place[];  // [warp][row of the range]: first the warp's tokens of the row, then where they go
  __shared__ int totals[kMaxRange];
  __shared__ int fold[kOrderWarps];
  __shared__ __align__(128) Zeros zeros;
  __shared__ int next_row, listing;  // the next row to look at for zeroing; warps that are still listing
  pdl_prologue();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t first_row = static_cast<int64_t>(blockIdx.x) * range;
  const int rows = static_cast<int>(min(static_cast<int64_t>(range), vocab - first_row));
  if (threadIdx.x == 0) {
    next_row = 0;
    listing = kListWarps;
  }
  zeros.clear(kOrderThreads);
  for (int i = threadIdx.x; i < kListWarps * range; i += kOrderThreads) place[i] = 0;
  __syncthreads();
  // the ids in one contiguous piece per warp, so that piece order is token order
  const int piece = (tokens + kListWarps - 1) / kListWarps;
  auto piece_start = [&](int p) { return static_cast<int>(min(static_cast<int64_t>(tokens), static_cast<int64_t>(p) * piece)); };
  const int begin = piece_start(warp), end = warp < kListWarps ? piece_start(warp + 1) : begin;
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
    for (int w = 0; w < kListWarps; ++w) {
      const int n = place[w * range + threadIdx.x];
      place[w * range + threadIdx.x] = mine;
      mine += n;
    }
    totals[threadIdx.x] = mine;
    hit[first_row + threadIdx.x] = mine != 0;
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
    for (int w = 0; w < kListWarps; ++w) place[w * range + threadIdx.x] += at;
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) {
    count[0] = start + all;
    count[1] = 0;  // the join kernel's next row to zero
  }
  __syncthreads();
  if (warp < kListWarps) {
    int* next = place + warp * range;
    for (int t0 = begin; t0 < end; t0 += 32 * AHEAD) {
      fetch(t0, end);
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
    if (lane == 0) atomicSub(&listing, 1);
  } else {
    for (;;) {
      int r = rows;
      if (lane == 0 && *static_cast<volatile int*>(&listing) > 0) r = atomicAdd(&next_row, kZeroRows);  // whichever warp takes them writes the same zeros
      r = __shfl_sync(0xffffffffu, r, 0);
      if (r >= rows) break;
      r += lane / kZeroLanes;
      if (r < rows && totals[r] == 0) zero_row(zeros, grad_weight + (first_row + r) * cols, cols);
      bulk_commit();
      bulk_wait_read<4>();  // no further ahead than that: the kernel ends with the list
    }
    bulk_wait_all<0>();
  }
  __syncthreads();
  if (threadIdx.x == 0) resume[blockIdx.x] = next_row;  // rows below it are done
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

// `fillers` of the CTAs zero the rows without tokens that the order kernel has not come to.  The others add up the parts of
// the runs that cross units.  A CTA looks after eight units, one per warp, and 256 columns; a warp has
// work where a run begins in its unit and goes on in the next.  A run of more than kLongRun parts is added up by all warps,
// each an equal share of its parts, the shares in warp order.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kJoinColumns = 256;
constexpr int kLongRun = 32;
constexpr int kJoinWords = kJoinColumns / 128;  // float4 of a lane: columns lane * 4 + 128 * i

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

// sum += the four columns from c of one part, for each of the lane's words
__device__ __forceinline__ void add_part(const float* part, int64_t cols, int64_t c0, float4 (&sum)[kJoinWords]) {
  float4 v[kJoinWords];
#pragma unroll
  for (int i = 0; i < kJoinWords; ++i) {
    const int64_t c = c0 + 128 * i;
    v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (cols % 4 == 0) {
      if (c < cols) v[i] = *reinterpret_cast<const float4*>(part + c);
    } else {
      if (c < cols) v[i].x = part[c];
      if (c + 1 < cols) v[i].y = part[c + 1];
      if (c + 2 < cols) v[i].z = part[c + 2];
      if (c + 3 < cols) v[i].w = part[c + 3];
    }
  }
#pragma unroll
  for (int i = 0; i < kJoinWords; ++i) sum[i].x += v[i].x, sum[i].y += v[i].y, sum[i].z += v[i].z, sum[i].w += v[i].w;
}
template <typename T>
__device__ __forceinline__ void put_row(T* out, int64_t cols, int64_t c0, const float4 (&sum)[kJoinWords], float scale) {
#pragma unroll
  for (int i = 0; i < kJoinWords; ++i) {
    const int64_t c = c0 + 128 * i;
    if (c < cols) out[c] = Num<T>::down(sum[i].x * scale);
    if (c + 1 < cols) out[c + 1] = Num<T>::down(sum[i].y * scale);
    if (c + 2 < cols) out[c + 2] = Num<T>::down(sum[i].z * scale);
    if (c + 3 < cols) out[c + 3] = Num<T>::down(sum[i].w * scale);
  }
}

template <typename T>
__global__ void __launch_bounds__(kJoinThreads, 3)
embedding_join_kernel(const int32_t* id, const int32_t* count, const float* parts, T* grad_weight, int unit, int capacity, int64_t cols, float scale, int fillers,
                      int column_tiles, const uint8_t* hit, const int32_t* resume, int* next_row, int64_t vocab, int range) {
  __shared__ int long_parts[kJoinWarps], long_run[kJoinWarps];  // of each warp's run, 0: it was short, or there was none
  __shared__ float4 share[kJoinWarps][kJoinWords][32];
  pdl_prologue();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x;
  if (b < fillers) {  // two of an SM's three places: eight rows of the table at a time and warp
    __shared__ __align__(128) Zeros zeros;
    zeros.clear(kJoinThreads);
    __syncthreads();
    for (;;) {
      int v0 = 0;
      if (lane == 0) v0 = atomicAdd(next_row, 2 * kZeroRows);  // whichever warp takes them writes the same zeros
      v0 = __shfl_sync(0xffffffffu, v0, 0);
      if (v0 >= vocab) break;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int64_t v = v0 + k * kZeroRows + lane / kZeroLanes;
        if (v < vocab && hit[v] == 0 && v % range >= resume[v / range]) zero_row(zeros, grad_weight + v * cols, cols);
      }
      bulk_commit();
      bulk_wait_read<4>();
    }
    bulk_wait_all<0>();
    return;
  }
  const int joiner = b - fillers, block = joiner / column_tiles;
  const int u = block * kJoinWarps + warp;
  const int64_t first = static_cast<int64_t>(u) * unit, c0 = static_cast<int64_t>(joiner % column_tiles) * kJoinColumns + lane * 4;
  // the ids around the unit's two ends and the length of the list, in one round of loads
  const int64_t at = lane == 0 ? first - 1 : lane == 1 ? first : first + unit + lane - 3;
  const int mine = lane < 4 && at >= 0 && at < capacity ? id[at] : -1;
  const int total = *count, units = (total + unit - 1) / unit;
  const int before = __shfl_sync(0xffffffffu, mine, 0), start = __shfl_sync(0xffffffffu, mine, 1), run = __shfl_sync(0xffffffffu, mine, 2), behind = __shfl_sync(0xffffffffu, mine, 3);
  int n = 0;  // parts: the second of unit u, the first of the units behind it
  if (first + unit < total && behind == run && (start != run || before != run)) {
    n = last_unit(id, run, u, units, unit) - u + 1;
    if (n <= kLongRun) {
      float4 sum[kJoinWords] = {};
      add_part(parts + (static_cast<int64_t>(u) * 2 + 1) * cols, cols, c0, sum);
#pragma unroll 4
      for (int i = 1; i < n; ++i) add_part(parts + static_cast<int64_t>(u + i) * 2 * cols, cols, c0, sum);
      put_row(grad_weight + run * cols, cols, c0, sum, scale);
    }
  }
  if (lane == 0) {
    long_parts[warp] = n > kLongRun ? n : 0;
    long_run[warp] = run;
  }
  __syncthreads();
  for (int k = 0; k < kJoinWarps; ++k) {
    n = long_parts[k];
    if (n == 0) continue;
    const int64_t begin = static_cast<int64_t>(block) * kJoinWarps + k;
    float4 sum[kJoinWords] = {};
#pragma unroll 4
    for (int i = static_cast<int>(static_cast<int64_t>(n) * warp / kJoinWarps); i < static_cast<int>(static_cast<int64_t>(n) * (warp + 1) / kJoinWarps); ++i)
      add_part(parts + ((begin + i) * 2 + (i == 0 ? 1 : 0)) * cols, cols, c0, sum);
#pragma unroll
    for (int i = 0; i < kJoinWords; ++i) share[warp][i][lane] = sum[i];
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int i = 0; i < kJoinWords; ++i) {
        sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < kJoinWarps; ++w) {
          const float4 v = share[w][i][lane];
          sum[i].x += v.x, sum[i].y += v.y, sum[i].z += v.z, sum[i].w += v.w;
        }
      }
      put_row(grad_weight + long_run[k] * cols, cols, c0, sum, scale);
    }
    __syncthreads();
  }
}

struct Scratch {
  int32_t *token, *id, *count, *resume;
  uint8_t* hit;
  float* parts;
};
// Sorted tokens per unit: long units mean few runs that cross them, as long as some 700 CTAs are left.
int unit_length(int64_t tokens, int64_t cols) {
  int unit = 8;
  while (unit < kMaxUnit && tokens * ceil_div(cols, 512) / (2 * unit) >= 700) unit *= 2;
  return unit;
}
// CTAs of the order kernel: one per SM, or as many as ranges of kMaxRange rows take.
constexpr int kMaxOrderCtas = 512;
int64_t order_ctas(int64_t vocab) { return std::max<int64_t>(std::min(sm_count(), kMaxOrderCtas), ceil_div(vocab, kMaxRange)); }
size_t scratch_layout(int64_t tokens, int64_t vocab, int64_t cols, char* base, Scratch* out) {
  const int64_t units = ceil_div(tokens, unit_length(tokens, cols));
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 15) / 16 * 16;
    return base + here;
  };
  Scratch s;
  s.count = reinterpret_cast<int32_t*>(take(8));
  s.resume = reinterpret_cast<int32_t*>(take(static_cast<size_t>(std::max<int64_t>(kMaxOrderCtas, ceil_div(vocab, kMaxRange))) * 4));
  s.hit = reinterpret_cast<uint8_t*>(take(static_cast<size_t>(vocab)));
  s.token = reinterpret_cast<int32_t*>(take(static_cast<size_t>(tokens) * 4));
  s.id = reinterpret_cast<int32_t*>(take(static_cast<size_t>(tokens) * 4));
  s.parts = reinterpret_cast<float*>(take(static_cast<size_t>(units) * 2 * static_cast<size_t>(cols) * 4));
  if (out != nullptr) *out = s;
  return at;
}

// The join kernel counts rows in 32 bits, and each of its 2 * 8 * (SMs) filling warps goes eight rows past the last one to find
// that it is done: room for that below 2^31, for up to 512 SMs.
constexpr int64_t kMaxVocab = (1LL << 31) - (1LL << 16);
int check_sizes(const char* fn, int64_t tokens, int64_t vocab, int64_t cols, int dtype) {
  if (!dtype_ok(dtype)) return fail(B200_ERR_DTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (tokens < 0 || vocab < 0 || cols < 0) return fail(B200_ERR_SHAPE, "%s: negative size", fn);
  if (tokens > (1LL << 30) || vocab > kMaxVocab) return fail(B200_ERR_SHAPE, "%s: tokens=%lld exceeds 2^30 or vocab=%lld 2^31-2^16", fn, (long long)tokens, (long long)vocab);
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
  const int range = static_cast<int>(ceil_div(vocab, order_ctas(vocab)));
  const size_t smem = static_cast<size_t>(range) * kListWarps * sizeof(int);
  constexpr auto order = embedding_order_kernel<T, I>;
  if (int rc = allow_smem<order, kMaxRange * kListWarps * static_cast<int>(sizeof(int))>("embedding_order_kernel")) return rc;
  const int pad = padding >= 0 && padding < vocab ? static_cast<int>(padding) : -1;
  launch(order, static_cast<unsigned>(ceil_div(vocab, range)), kOrderThreads, smem, st, static_cast<const I*>(ids), static_cast<int>(tokens), vocab, pad,
         range, s.token, s.id, s.count, s.hit, s.resume, out, cols);
  if (int rc = after_launch("embedding_order_kernel")) return rc;
  const int unit = unit_length(tokens, cols);
  const int64_t words = vec ? cols / V : cols, units = ceil_div(tokens, unit);
  if (tokens > 0) {
    const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(ceil_div(words, kSumThreads)));
    if (vec)
      launch(embedding_sum_kernel<T, true>, grid, kSumThreads, 0, st, g, s.token, s.id, s.count, out, s.parts, unit, static_cast<int>(tokens), words, cols, ldg, scale);
    else
      launch(embedding_sum_kernel<T, false>, grid, kSumThreads, 0, st, g, s.token, s.id, s.count, out, s.parts, unit, static_cast<int>(tokens), words, cols, ldg, scale);
    if (int rc = after_launch("embedding_sum_kernel")) return rc;
  }
  const int fillers = 2 * sm_count();
  const int64_t tiles = ceil_div(cols, kJoinColumns), joins = units > 1 ? ceil_div(units - 1, kJoinWarps) * tiles : 0;
  launch(embedding_join_kernel<T>, static_cast<unsigned>(fillers + joins), kJoinThreads, 0, st, s.id, s.count, static_cast<const float*>(s.parts), out, unit,
         static_cast<int>(tokens), cols, scale, fillers, static_cast<int>(tiles), static_cast<const uint8_t*>(s.hit), static_cast<const int32_t*>(s.resume), s.count + 1, vocab, range);
  return after_launch("embedding_join_kernel");
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
  *bytes = scratch_layout(tokens, vocab, cols, nullptr, nullptr);
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
  const size_t need = scratch_layout(tokens, vocab, cols, static_cast<char*>(scratch), &s);
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
