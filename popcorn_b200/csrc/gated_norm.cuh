// Shared by the two directions of the gated residual norm (gated_norm.cu, gated_norm_backward.cu).
#pragma once

#include <algorithm>
#include <initializer_list>

#include "activations.cuh"
#include "common.cuh"
#include "tma.cuh"

namespace b200 {
namespace {

enum Activation { kIdentity = 0, kTanh = 1, kSigmoid = 2 };

// One load: a 128-bit word of T, or where width, strides or pointers do not allow words, two neighbouring elements at once, or
// where they do not allow that either, one element.
enum Access { kWords = 0, kPairs = 1, kSingles = 2 };
template <typename T, int ACCESS>
struct Word;
template <typename T>
struct Word<T, kWords> {
  static constexpr int N = Num<T>::kVec;
  using Raw = uint4;
  static __device__ __forceinline__ Raw zero() { return make_uint4(0, 0, 0, 0); }
  static __device__ __forceinline__ Raw load(const T* p) { return ld_stream(p); }
  static __device__ __forceinline__ Raw load_shared_by_rows(const T* p) { return ld_kept(p); }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[N]) { Num<T>::unpack(r, f); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[N]) { st_stream(p, Num<T>::pack(f)); }
};
template <typename T>
struct Word<T, kPairs> {
  static constexpr int N = 2;
  struct alignas(2 * sizeof(T)) Raw {
    T lo, hi;
  };
  static __device__ __forceinline__ Raw zero() { return {Num<T>::down(0.f), Num<T>::down(0.f)}; }
  static __device__ __forceinline__ Raw load(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ Raw load_shared_by_rows(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[2]) { f[0] = Num<T>::up(r.lo), f[1] = Num<T>::up(r.hi); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[2]) { *reinterpret_cast<Raw*>(p) = {Num<T>::down(f[0]), Num<T>::down(f[1])}; }
};
template <typename T>
struct Word<T, kSingles> {
  static constexpr int N = 1;
  using Raw = T;
  static __device__ __forceinline__ Raw zero() { return Num<T>::down(0.f); }
  static __device__ __forceinline__ Raw load(const T* p) { return *p; }
  static __device__ __forceinline__ Raw load_shared_by_rows(const T* p) { return *p; }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[1]) { f[0] = Num<T>::up(r); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[1]) { *p = Num<T>::down(f[0]); }
};

// tanh below 1/4: the next term of its series is below 1e-8 of it (a NaN is not below 1/4 and is kept by the sigmoid)
__device__ __forceinline__ float tanh_series(float g) {
  const float q = g * g;
  return g * fmaf(q, fmaf(q, fmaf(q, fmaf(q, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
}
// 16-bit types: the approximate exponential and reciprocal of activations.cuh, off by some 1e-6 of the value where T rounds
// by 2^-11 at best; the gate of every row of [16376, 5120] fp16 costs 166 us with tanhf, 152 with this.  fp32: CUDA's own.
template <typename T>
__device__ __forceinline__ float activate(float g, int act) {
  if (act == kIdentity) return g;
  if constexpr (sizeof(T) == 4) return act == kTanh ? tanhf(g) : __fdiv_rn(1.f, __fadd_rn(1.f, expf(-g)));
  const float h = act == kTanh ? 2.f * g : g;
  const float sigmoid = sigmoid_f32<1>(h);
  if (act == kSigmoid) return sigmoid;
  const float series = tanh_series(g);
  return fabsf(g) < 0.25f ? series : fmaf(2.f, sigmoid, -1.f);  // where it cancels, the series
}
// d act / d g from the activation's value
__device__ __forceinline__ float activation_slope(float value, int act) {
  if (act == kTanh) return __fsub_rn(1.f, __fmul_rn(value, value));
  if (act == kSigmoid) return __fmul_rn(value, __fsub_rn(1.f, value));
  return 1.f;
}

// 1 / sqrt(sum of squares / cols + eps), within two units in the last place (nothing is rounded to T in between)
__device__ __forceinline__ float inv_rms(float sumsq, float inv_cols, float eps) { return rsqrtf(fmaf(sumsq, inv_cols, eps)); }

// A sum over the TPR threads of a row, TPR a power of two.  Up to a warp: shuffles.  Wider: one barrier
// (rows wider than a warp have the CTA to themselves); `slot` is shared memory that no thread still reads from an earlier
// call.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* slot) {
  v = warp_sum(v);
  if constexpr (TPR > 32) {
    constexpr int WARPS = TPR / 32;
    const int lane = threadIdx.x & 31;
    if (lane == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    v = slot[lane & (WARPS - 1)];
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
  }
  return v;
}
// Four at once: two steps leave each lane with a quarter of the lanes' sum of one value (value 2 (lane / 8 % 2) + lane / 16),
// so six exchanges do for four sums, where one after the other takes twenty.
template <int TPR>
__device__ __forceinline__ void row_sums(float (&v)[4], float (*slot)[16]) {
  const int lane = threadIdx.x & 31;
  const bool high = lane & 16, odd = lane & 8;
  const float v01 = (high ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, high ? v[0] : v[1], 16);
  const float v23 = (high ? v[3] : v[2]) + __shfl_xor_sync(0xffffffffu, high ? v[2] : v[3], 16);
  float sum = (odd ? v23 : v01) + __shfl_xor_sync(0xffffffffu, odd ? v01 : v23, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if constexpr (TPR > 32) {
    constexpr int WARPS = TPR / 32;
    if ((lane & 7) == 0) slot[(odd ? 2 : 0) + (high ? 1 : 0)][threadIdx.x >> 5] = sum;
    __syncthreads();
    const float* mine = slot[(odd ? 2 : 0) + (high ? 1 : 0)];
    sum = mine[lane & (WARPS < 8 ? WARPS - 1 : 7)];
    if constexpr (WARPS == 16) sum += mine[8 + (lane & 7)];
#pragma unroll
    for (int o = WARPS < 8 ? WARPS / 2 : 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  v[0] = __shfl_sync(0xffffffffu, sum, 0);
  v[1] = __shfl_sync(0xffffffffu, sum, 16);
  v[2] = __shfl_sync(0xffffffffu, sum, 8);
  v[3] = __shfl_sync(0xffffffffu, sum, 24);
}

// ------------------------------------------------------------------- ring --
//
// The rows of a walker in shared memory.  Arrays of rows (x, residual, ...) take turns: row r of array a is copy
// r * arrays + a, in slot (r * arrays + a) % slots, so any number of slots above `arrays` keeps copies in flight.  The
// copies of a row complete one barrier, barrier r % rows_ahead.  A thread for each array issues them; a slot is filled
// again once the walker is past a barrier behind its last read.
// Every wait is bounded.  A thread whose wait runs out fetches what it reads of that row with ordinary loads (a copy that
// lands beside them brings the same data) and leaves the row's number in `broken`.  Behind the row's next barrier all
// threads see it and agree: nothing is issued any more, the copies in flight are waited for, bounded again, and the
// remaining rows are fetched with ordinary loads, into slots that no copy can reach.  Should that second wait run out as
// well, a late copy could: the remaining rows, if in words, give NaN.
// A bulk copy moves multiples of 16 bytes between 16-byte boundaries: of a row that starts or ends elsewhere the ring
// holds what lies between, [lo, hi) in bytes from the row's start, and the few elements around it are loaded directly.
constexpr int kMaxSlots = 16;

__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A row of one array as a thread reads it
struct RowView {
  uint32_t memory;  // shared-memory address of the row's first byte (where it would be, for a row off the boundaries)
  uint32_t lo, hi;  // unused for rows in words
  const void* row;
};

template <typename T, bool VEC, int TPR>
struct Ring {
  uint32_t full, memory;  // shared-memory addresses
  uint32_t broken;  // shared-memory address of 0, or 1 + the row (from the walker's first) whose wait ran out; behind it: 1, the wait for the rest did too
  int count, slots, rows_ahead;
  uint32_t row_bytes, slot_bytes;
  // the issuing threads (the first `count` of the walker, one array each): their array and the next row of it
  const T* base;
  int64_t ld;
  uint32_t put_row, first_row, last_row;
  int64_t put_copy;  // of the next row of this array
  int put, put_bar;  // its slot and barrier
  int take, take_bar;
  uint32_t phase;

  // memory: slots * slot_bytes of this walker; all threads of the CTA call this.  array(a, base, ld) names the rows of array a.
  template <typename Arrays>
  __device__ __forceinline__ void start(uint64_t* barriers, unsigned char* mem, uint32_t (&flags)[2], int n, uint32_t bytes, uint32_t padded, uint32_t first, uint32_t last, int arrays,
                                        Arrays&& array) {
    full = smem_addr(barriers), memory = smem_addr(mem), broken = smem_addr(flags);
    count = arrays, slots = n, row_bytes = bytes, slot_bytes = padded, put_row = first_row = first, last_row = last;
    rows_ahead = (slots + count - 1) / count;  // a barrier is used again only after the row before was given free
    put_copy = put = threadIdx.x;
    put_bar = take = take_bar = 0, phase = 0;
    array(static_cast<int>(threadIdx.x), base, ld);
    if (threadIdx.x == 0) {
      flags[0] = flags[1] = 0;
      for (int k = 0; k < rows_ahead; ++k) mbar_init(barriers + k, count);
      mbar_init_fence();
    }
    __syncthreads();
    if (threadIdx.x < count) issue(slots);
  }
  // bytes of a row that the ring holds, from the row's start
  __device__ __forceinline__ void span(const T* row, uint32_t& lo, uint32_t& hi) const {
    if constexpr (VEC) {
      lo = 0, hi = row_bytes;
    } else {
      const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row)) & 15u;
      lo = (16u - at) & 15u;
      hi = at + row_bytes < 16u ? 0u : ((at + row_bytes) & ~15u) - at;
      if (hi < lo) hi = lo;
    }
  }
  // an issuing thread: its array's copies below `limit`
  __device__ __forceinline__ void issue(int64_t limit) {
    for (; put_copy < limit && put_row < last_row; put_copy += count, ++put_row) {
      const T* row = base + put_row * ld;
      uint32_t lo, hi;
      span(row, lo, hi);
      const uint32_t bar = full + put_bar * 8;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(hi - lo) : "memory");
      if (hi > lo)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(memory + put * slot_bytes),
                     "l"(reinterpret_cast<const unsigned char*>(row) + lo), "r"(hi - lo), "r"(bar)
                     : "memory");
      put += count;
      if (put >= slots) put -= slots;
      if (++put_bar == rows_ahead) put_bar = 0;
    }
  }
  static __device__ __forceinline__ uint32_t read_flag(uint32_t at) {
    uint32_t v;
    asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
  }
  static __device__ __forceinline__ void write_flag(uint32_t at, uint32_t v) { asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
  // All threads, past a barrier behind the wait for row `row`, with `free` rows read for the last time: their slots go to the next rows.
  __device__ __forceinline__ void release(uint32_t row, uint32_t free) {
    if (threadIdx.x >= count) return;
    const uint32_t at = read_flag(broken);  // a thread that is ahead may have left the next row's number: that counts behind its barrier
    if (at == 0 || at > row + 1) issue(static_cast<int64_t>(free) * count + slots);
  }
  // Have all copies landed that were issued with `free` rows given free, those from row `row` on among them?  put: the next row of
  // this thread's array, `rows` or above if it issues none.  A call: the registers of the loop around are not to make room for it.
  static __device__ __noinline__ bool drain(uint32_t full, int count, int slots, int rows_ahead, uint32_t put, uint32_t rows, uint32_t row, uint32_t free) {
    rows = static_cast<uint32_t>(min((static_cast<int64_t>(free) * count + slots + count - 1) / count, static_cast<int64_t>(rows)));  // of which a copy was issued
    for (; put < rows; ++put) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(full + put % rows_ahead * 8) : "memory");  // the last one's other arrays: without a copy
    bool landed = true;
    for (; row < rows; ++row) landed = wait_for(full + row % rows_ahead * 8, row / rows_ahead & 1u, kSpinLimit) && landed;
    return landed;
  }
  static __device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, uint32_t limit) {
    for (uint32_t i = 0; i < limit; ++i) {
      uint32_t done;
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(done)
          : "r"(bar), "r"(parity)
          : "memory");
      if (done) return true;
    }
    atomicAdd(&g_wait_timeouts, 1u);
    return false;
  }
  // the next row in turn, row `row` from the walker's first: has it landed?  late: rows are given free at their own end, else at the
  // first barrier of the row behind them
  __device__ __forceinline__ bool wait(uint32_t row, uint32_t probes, bool late) {
    const uint32_t at = read_flag(broken);
    bool landed = at == 0 || at > row;
    if (landed) {
      landed = wait_for(full + take_bar * 8, phase, probes);
      if (!landed) write_flag(broken, row + 1);
    } else if (at == row) {  // the row before was the broken one, and the last given free were those before it
      const uint32_t rows = last_row - first_row;
      if (!drain(full, count, slots, rows_ahead, threadIdx.x < count ? put_row - first_row : rows, rows, row - 1, late ? row - 1 : row < 2 ? 0 : row - 2)) write_flag(broken + 4, 1);
    }
    if (++take_bar == rows_ahead) {
      take_bar = 0;
      phase ^= 1;
    }
    return landed;
  }
  // a row that has not landed: may a late copy reach its words?
  __device__ __forceinline__ bool unsound() const { return VEC && read_flag(broken + 4) != 0; }
  // its arrays one after the other, starting with array 0: row `row` of the array at `from`
  __device__ __forceinline__ RowView view(const T* from, int64_t stride, uint32_t row, bool landed) {
    RowView v;
    v.memory = memory + take * slot_bytes;
    if (++take == slots) take = 0;
    if constexpr (VEC) {
      if (!landed) {
        const unsigned char* bytes = reinterpret_cast<const unsigned char*>(from + row * stride);
        for (uint32_t at = (threadIdx.x) * 16u; at < row_bytes; at += TPR * 16u) st_shared(v.memory + at, ld_stream(bytes + at));
      }
    } else {
      v.row = from + row * stride;
      span(from + row * stride, v.lo, v.hi);
      v.memory -= v.lo;
      if (!landed) v.lo = v.hi = 0;
    }
    return v;
  }
  // Behind the last row: nothing is in flight, unless it was the one whose wait ran out.
  __device__ __forceinline__ void finish() const {
    const uint32_t rows = last_row - first_row;
    if (rows > 0 && read_flag(broken) == rows) (void)wait_for(full + (rows - 1) % rows_ahead * 8, (rows - 1) / rows_ahead & 1u, kSpinLimit);
  }
};

__device__ __forceinline__ uint32_t range_start(uint32_t rows, int walkers, int walker) {
  return static_cast<uint32_t>(static_cast<uint64_t>(rows) * walker / walkers);
}

// What a thread of a walker loads at a time, as fp32 pairs (two elements per instruction): a 128-bit word, or two neighbouring
// elements, together where all rows allow it (RowShape::pairs), else one after the other, the second perhaps behind the row.
struct RowShape {
  int cols;
  bool pairs;
};
template <typename T, bool VEC>
struct Pairs {
  static constexpr int P = Num<T>::kVec / 2, N = 2 * P;
  static __device__ __forceinline__ void unpack(const uint4& raw, Float2x (&out)[P]) {
    float f[N];
    Num<T>::unpack(raw, f);
#pragma unroll
    for (int j = 0; j < P; ++j) out[j] = pack_f2(f[2 * j], f[2 * j + 1]);
  }
  static __device__ __forceinline__ void load(const RowView& v, int w, RowShape, Float2x (&out)[P]) { unpack(ld_shared(v.memory + w * 16), out); }
  static __device__ __forceinline__ void load_shared_by_rows(const T* row, int w, RowShape, Float2x (&out)[P]) { unpack(ld_kept(row + w * N), out); }
  static __device__ __forceinline__ void store(T* row, int w, RowShape, const Float2x (&v)[P]) {
    float f[N];
#pragma unroll
    for (int j = 0; j < P; ++j) unpack_f2(v[j], f[2 * j], f[2 * j + 1]);
    st_stream(row + w * N, Num<T>::pack(f));
  }
};
template <typename T>
struct Pairs<T, false> {
  static constexpr int P = 1, N = 2;
  static __device__ __forceinline__ float element(const RowView& v, uint32_t c) {
    const uint32_t byte = c * static_cast<uint32_t>(sizeof(T));
    if (byte < v.lo || byte >= v.hi) return Num<T>::up(static_cast<const T*>(v.row)[c]);
    if constexpr (sizeof(T) == 4) {
      float f;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(v.memory + byte) : "memory");
      return f;
    } else {
      uint16_t bits;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(v.memory + byte) : "memory");
      return Num<T>::up(*reinterpret_cast<const T*>(&bits));
    }
  }
  using Two = Word<T, kPairs>;
  static __device__ __forceinline__ Float2x as_pair(const typename Two::Raw& raw) {
    float f[2];
    Two::unpack(raw, f);
    return pack_f2(f[0], f[1]);
  }
  static __device__ __forceinline__ void load(const RowView& v, int w, RowShape shape, Float2x (&out)[1]) {
    if (shape.pairs) {
      const uint32_t byte = static_cast<uint32_t>(w) * 2 * static_cast<uint32_t>(sizeof(T));
      if (byte < v.lo || byte >= v.hi) {
        out[0] = as_pair(Two::load(static_cast<const T*>(v.row) + 2 * w));
      } else if constexpr (sizeof(T) == 4) {
        float lo, hi;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(lo), "=f"(hi) : "r"(v.memory + byte) : "memory");
        out[0] = pack_f2(lo, hi);
      } else {
        uint32_t bits;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(bits) : "r"(v.memory + byte) : "memory");
        out[0] = as_pair(*reinterpret_cast<const typename Two::Raw*>(&bits));
      }
      return;
    }
    out[0] = pack_f2(element(v, 2 * w), 2 * w + 1 < shape.cols ? element(v, 2 * w + 1) : 0.f);
  }
  static __device__ __forceinline__ void load_shared_by_rows(const T* row, int w, RowShape shape, Float2x (&out)[1]) {
    out[0] = pack_f2(Num<T>::up(row[2 * w]), 2 * w + 1 < shape.cols ? Num<T>::up(row[2 * w + 1]) : 0.f);
  }
  static __device__ __forceinline__ void store(T* row, int w, RowShape shape, const Float2x (&v)[1]) {
    float f[2];
    unpack_f2(v[0], f[0], f[1]);
    if (shape.pairs) {
      Two::store(row + 2 * w, f);
      return;
    }
    row[2 * w] = Num<T>::down(f[0]);
    if (2 * w + 1 < shape.cols) row[2 * w + 1] = Num<T>::down(f[1]);
  }
};
__device__ __forceinline__ Float2x both(float v) { return pack_f2(v, v); }
__device__ __forceinline__ float pair_total(Float2x v) {
  float lo, hi;
  unpack_f2(v, lo, hi);
  return __fadd_rn(lo, hi);
}
template <typename T>
__device__ __forceinline__ Float2x activate2(Float2x g, int act) {
  float lo, hi;
  unpack_f2(g, lo, hi);
  return pack_f2(activate<T>(lo, act), activate<T>(hi, act));
}

// The activation of a row's own gate in the backward, without a branch per element: tanh and the sigmoid as one expression of
// sigma(in * g), off by some 3e-7 of the value for every type.  With the branches of activate() the backward of bf16
// [16384, 4096] with a tanh gate per row takes 385 us, with this 313; the forward, which has fewer registers, is slower with
// it ([4095, 2050] fp32 55 us against 47).
struct RowAct {
  float in, out, shift, series;  // |g| below `series`: tanh_series
  int kind;
};
__device__ __forceinline__ RowAct make_row_act(int kind) { return kind == kTanh ? RowAct{2.f, 2.f, -1.f, 0.25f, kind} : RowAct{1.f, 1.f, 0.f, -1.f, kind}; }
template <int P>
__device__ __forceinline__ void activate_row(Float2x (&g)[P], const RowAct& act) {
  if (act.kind == kIdentity) return;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    float v[2];
    unpack_f2(g[j], v[0], v[1]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float value = fmaf(act.out, sigmoid_f32<1>(act.in * v[k]), act.shift);
      v[k] = fabsf(v[k]) < act.series ? tanh_series(v[k]) : value;
    }
    g[j] = pack_f2(v[0], v[1]);
  }
}
// d act / d g from the value: 1 - v^2, v - v^2 or 1
__device__ __forceinline__ float row_slope(float value, const RowAct& act) { return act.kind == kIdentity ? 1.f : fmaf(-value, value, act.kind == kTanh ? 1.f : value); }

constexpr int kColumns = 16;  // columns per thread of a walker
constexpr int kMaxWalk = 512;
constexpr int kWalkColumns = kMaxWalk * kColumns;
constexpr int kRingBytes = 196 * 1024;  // of an SM; the rest of its 228 KB is what 16 CTAs need besides

// s of one element, for the kernels that go over a row more than once
__device__ __forceinline__ float stream_value(float x, float residual, float factor, float r1, float residual_scale) {
  return fmaf(r1 * factor, x, residual_scale * residual);
}
// scale * act(gate) * (post_weight + offset) of one column
template <typename T>
__device__ __forceinline__ float branch_factor(const T* post, const T* gate_row, int64_t c, float offset, float scale, int act) {
  float f = scale;
  if (gate_row != nullptr) f *= activate<T>(Num<T>::up(gate_row[c]), act);
  if (post != nullptr) f *= Num<T>::up(post[c]) + offset;
  return f;
}

// The threads of a walker for a row of `cols`, its rows' slots in shared memory, and how many walkers share `rows`: as many
// as give an SM 512 threads of 128 registers.
struct WalkPlan {
  int tpr, walkers, slots;
  uint32_t slot_bytes;
};
WalkPlan plan_walk(int64_t rows, int64_t cols, size_t element) {
  WalkPlan p;
  p.tpr = 32;
  while (p.tpr * kColumns < cols) p.tpr *= 2;
  const int per_sm = kMaxWalk / p.tpr;
  p.walkers = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rows, static_cast<int64_t>(sm_count()) * per_sm)));
  p.slot_bytes = static_cast<uint32_t>(std::max<int64_t>(1, ceil_div(cols * static_cast<int64_t>(element), 16)) * 16);
  p.slots = static_cast<int>(std::min<size_t>(kMaxSlots, kRingBytes / per_sm / p.slot_bytes));  // at least 6: a row's arrays, five at most, fit
  return p;
}

// The widest access that the width, the strides and the pointers of all operands (NULL: none) allow.
Access access_of(size_t element, int64_t cols, std::initializer_list<const void*> pointers, std::initializer_list<int64_t> strides) {
  for (const Access access : {kWords, kPairs}) {
    const int64_t elements = access == kWords ? 16 / static_cast<int64_t>(element) : 2;
    bool fits = cols % elements == 0;
    for (const void* p : pointers) fits = fits && aligned(p, elements * element);
    for (const int64_t ld : strides) fits = fits && ld % elements == 0;
    if (fits) return access;
  }
  return kSingles;
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
