// Balance loss of the MoE router, its z-loss and the per-expert counts, with the gradient of both losses.
//
// Tokens t with logits l_t, p_t = softmax(l_t), lse_t = log sum exp(l_t), k picks each; groups g (one, or one for each
// sequence), n_g tokens of a group that the mask keeps, n of all groups together, G the groups with n_g > 0:
//   f_ge = experts counts_ge / (k n_g),  P_ge = sum_t p_te / n_g
//   balance = 1/G sum_g sum_e f_ge P_ge,   z = 1/n sum_t lse_t^2
//   d balance / d l_te = p_te (f_ge - sum_j p_tj f_gj) / (G n_g)   (the counts carry no gradient)
//   d z / d l_te = 2 lse_t p_te / n
//
// Bound: HBM.  Forward: the logits and picks read once (a softmax row lives in the registers of a few lanes), every CTA
// leaves one line of sums, a second small kernel adds the lines up in a fixed order in fp64 (a cluster per group, each CTA
// some of the experts).  Backward: the logits read again, the gradient written; row maximum and sum come from the forward
// pass (8 bytes a token).  A lane has eight loads in flight, of one token or of several: with two, [131072, 256] fp32 took
// 91 us forward instead of 36.
#include <algorithm>
#include <type_traits>

#include "activations.cuh"
#include "common.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;

// WPL loads per lane, LPT lanes per token: lane l of a token holds loads l, l + LPT, ...
template <typename T, bool VEC>
struct Load;
template <typename T>
struct Load<T, true> {
  static constexpr int N = Num<T>::kVec;
  using Raw = uint4;
  static __device__ __forceinline__ Raw lowest() {  // -inf throughout
    const uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    return make_uint4(w, w, w, w);
  }
  static __device__ __forceinline__ Raw get(const T* p) { return ld_stream(p); }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[N]) { Num<T>::unpack(r, f); }
  static __device__ __forceinline__ void put(T* p, const float (&f)[N]) { st_stream(p, Num<T>::pack(f)); }
};
template <typename T>
struct Load<T, false> {
  static constexpr int N = 1;
  using Raw = T;
  static __device__ __forceinline__ Raw lowest() { return Num<T>::down(-INFINITY); }
  static __device__ __forceinline__ Raw get(const T* p) { return *p; }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[1]) { f[0] = Num<T>::up(r); }
  static __device__ __forceinline__ void put(T* p, const float (&f)[1]) { *p = Num<T>::down(f[0]); }
};

template <int LPT>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int LPT>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One line of sums per CTA, [groups][chunks] lines of each kind in scratch.
struct Partials {
  float* probs;   // [line][experts]
  int* picks;     // [line][experts]
  float* z;       // [line]
  int* kept;      // [line]
  double* group;  // [groups][3]: balance, z and tokens of a group
};

struct Shape {
  int64_t tokens, ld;  // tokens of a group
  int experts, top_k, chunks;
};
// CTA c of a group's `chunks` takes every chunks-th tile of tokens from tile c on: a padded tail is spread over all of them.

// exp(v - top): the hardware's power of two, off by 2^-22 and by 2^-24 of v - top (nothing for the largest terms of a row)
__device__ __forceinline__ float exp_from(float v, float top) { return ex2_approx(__fmul_rn(__fsub_rn(v, top), 1.4426950408889634f)); }

// WPL loads per lane of a token, LPT lanes per token, U tokens at a time
template <typename T, bool VEC, int LPT, int WPL, int U>
__global__ void __launch_bounds__(kThreads, 2)
balance_sums_kernel(const T* logits, const int32_t* indices, const uint8_t* mask, float2* stats, const Shape s, const Partials out) {
  using L = Load<T, VEC>;
  constexpr int N = L::N;
  constexpr int TOKENS = 32 / LPT;  // tokens of a warp side by side
  constexpr int WARPS = kThreads / 32;
  pdl_prologue();
  __shared__ int picks[kMaxExperts];
  __shared__ float fold[WARPS][LPT * WPL * N];
  __shared__ float fold_z[WARPS];
  __shared__ int fold_n[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lane_in_token = lane % LPT;
  const int64_t group = blockIdx.y, base = group * s.tokens;
  const int tokens = static_cast<int>(s.tokens);
  logits += base * s.ld;
  indices += base * s.top_k;
  if (mask != nullptr) mask += base;
  if (stats != nullptr) stats += base;
  for (int e = threadIdx.x; e < s.experts; e += kThreads) picks[e] = 0;
  __syncthreads();
  float sums[WPL][N], z = 0.f;
  int kept = 0;
#pragma unroll
  for (int i = 0; i < WPL; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) sums[i][j] = 0.f;
  // every lane of a warp runs the same number of iterations: the shuffles need them all
  constexpr int TILE = WARPS * TOKENS * U;
  // which of the next tile's tokens count: a tile ahead, so that the logits do not wait for the mask
  bool kept_next[U];
  auto look = [&](int64_t tile) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = tile * TILE + (warp * U + u) * TOKENS + lane / LPT;
      kept_next[u] = t < tokens && (mask == nullptr || mask[t] != 0);
    }
  };
  // loads behind the last expert are never made and stay -inf; those of a token that does not count are stale and not used
  typename L::Raw raw[U][WPL];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < WPL; ++i) raw[u][i] = L::lowest();
  look(blockIdx.x);
  for (int64_t tile = blockIdx.x; tile * TILE < tokens; tile += s.chunks) {
    const int t0 = static_cast<int>(tile) * TILE + warp * TOKENS * U;
    bool keep[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * TOKENS + lane / LPT;
      keep[u] = kept_next[u];
#pragma unroll
      for (int i = 0; i < WPL; ++i) {
        const int e = (lane_in_token + i * LPT) * N;
        if (keep[u] && e < s.experts) raw[u][i] = L::get(logits + t * s.ld + e);
      }
    }
    look(tile + s.chunks);
    // the tile's picks, their latency hidden behind that of the logits
    const int pick0 = static_cast<int>(tile) * TILE * s.top_k, pick_end = min(static_cast<int>(tile) * TILE + TILE, tokens) * s.top_k;
    for (int i0 = pick0 + threadIdx.x; i0 < pick_end; i0 += 4 * kThreads) {
      int e[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + k * kThreads;
        e[k] = i < pick_end ? indices[i] : -1;
        if (mask != nullptr && i < pick_end && mask[static_cast<unsigned>(i) / static_cast<unsigned>(s.top_k)] == 0) e[k] = -1;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (static_cast<unsigned>(e[k]) < static_cast<unsigned>(s.experts)) atomicAdd(&picks[e[k]], 1);  // whole numbers: any order
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[WPL][N], top = -INFINITY;
#pragma unroll
      for (int i = 0; i < WPL; ++i) {
        L::unpack(raw[u][i], v[i]);
#pragma unroll
        for (int j = 0; j < N; ++j) top = fmaxf(top, v[i][j]);
      }
      top = lanes_max<LPT>(top);
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < WPL; ++i) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          v[i][j] = exp_from(v[i][j], top);  // a row of -inf alone is NaN, as in a softmax
          total += v[i][j];
        }
      }
      total = lanes_sum<LPT>(total);
      if (keep[u]) {
        const float inv = __frcp_rn(total);
#pragma unroll
        for (int i = 0; i < WPL; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j) sums[i][j] = fmaf(v[i][j], inv, sums[i][j]);
        if (lane_in_token == 0) {
          const float lse = top + logf(total);
          z = fmaf(lse, lse, z);
          ++kept;
          if (stats != nullptr) stats[t0 + u * TOKENS + lane / LPT] = make_float2(top, total);
        }
      }
    }
  }
  // the lanes of a warp that hold the same experts, then the warps in order
#pragma unroll
  for (int o = LPT; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < WPL; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) sums[i][j] += __shfl_xor_sync(0xffffffffu, sums[i][j], o);
  }
  z = lanes_sum<32>(z);
  kept = __reduce_add_sync(0xffffffffu, kept);
  if (lane < LPT) {
#pragma unroll
    for (int i = 0; i < WPL; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) fold[warp][(lane + i * LPT) * N + j] = sums[i][j];
  }
  if (lane == 0) {
    fold_z[warp] = z;
    fold_n[warp] = kept;
  }
  __syncthreads();
  const int64_t line = group * s.chunks + blockIdx.x;
  for (int e = threadIdx.x; e < s.experts; e += kThreads) {
    float p = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) p += fold[w][e];
    out.probs[line * s.experts + e] = p;
    out.picks[line * s.experts + e] = picks[e];
  }
  if (threadIdx.x == 0) {
    float total = 0.f;
    int n = 0;
    for (int w = 0; w < WARPS; ++w) {
      total += fold_z[w];
      n += fold_n[w];
    }
    out.z[line] = total;
    out.kept[line] = n;
  }
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// table: f [groups][experts], then 1 / (G n_g) [groups], then 1 / n: what the backward multiplies with.
// A cluster per group adds up its lines: each CTA takes 32 experts at a time (the lanes of its warps; a warp every
// kGroupWarps-th line), and the first CTA adds up the CTAs' parts of the loss.
constexpr int kGroupThreads = 1024, kGroupWarps = kGroupThreads / 32;
constexpr int kMaxCluster = 8;
__device__ void write_totals(double balance, double z, double kept, int used, float* loss, float* z_loss) {
  *loss = used > 0 ? static_cast<float>(balance / used) : 0.f;
  *z_loss = kept > 0 ? static_cast<float>(z / kept) : 0.f;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__global__ void __launch_bounds__(kGroupThreads)
balance_group_kernel(const Shape s, const Partials in, int groups, int cluster, int32_t* counts, float* table, float* loss, float* z_loss) {
  pdl_prologue();
  __shared__ double fold_p[kGroupWarps][33];
  __shared__ int fold_c[kGroupWarps][33];
  __shared__ double fold_z[kGroupWarps];
  __shared__ long long fold_n[kGroupWarps];
  __shared__ double part;  // of the loss, of this CTA's experts
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = blockIdx.x % cluster;
  const int64_t group = blockIdx.x / cluster, line0 = group * s.chunks;
  double z = 0.0;
  long long n = 0;
  for (int c = threadIdx.x; c < s.chunks; c += kGroupThreads) {
    z += in.z[line0 + c];
    n += in.kept[line0 + c];
  }
  double balance = 0.0;  // of each warp's first lane
  for (int e0 = rank * 32; e0 < s.experts; e0 += cluster * 32) {
    const int e = e0 + lane;
    double p = 0.0;
    int picks = 0;
    constexpr int BATCH = 5;  // loads of either kind in flight
    for (int c0 = warp; c0 < s.chunks; c0 += BATCH * kGroupWarps) {
      float probs[BATCH];
      int counted[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int c = c0 + k * kGroupWarps;
        const bool there = c < s.chunks && e < s.experts;
        probs[k] = there ? in.probs[(line0 + c) * s.experts + e] : 0.f;
        counted[k] = there ? in.picks[(line0 + c) * s.experts + e] : 0;
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        p += probs[k];
        picks += counted[k];
      }
    }
    __syncthreads();  // the round before has been read
    fold_p[warp][lane] = p;
    fold_c[warp][lane] = picks;
    if (e0 == rank * 32) {  // here, and not before the first loads were asked for
      z = warp_sum_f64(z);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
      if (lane == 0) {
        fold_z[warp] = z;
        fold_n[warp] = n;
      }
    }
    __syncthreads();
    // warp w adds up what the warps have of expert w of the 32
    p = warp_sum_f64(fold_p[lane][warp]);
    picks = __reduce_add_sync(0xffffffffu, fold_c[lane][warp]);
    n = fold_n[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (lane == 0 && e0 + warp < s.experts) {
      const double kept = static_cast<double>(n), f = n > 0 ? static_cast<double>(picks) * s.experts / (kept * s.top_k) : 0.0;
      counts[group * s.experts + e0 + warp] = picks;
      table[group * s.experts + e0 + warp] = static_cast<float>(f);
      if (n > 0) balance += f * p / kept;
    }
  }
  __syncthreads();
  if (lane == 0) fold_p[0][warp] = balance;
  __syncthreads();
  if (warp == 0) {
    balance = warp_sum_f64(fold_p[0][lane]);
    if (lane == 0) part = balance;
  }
  cluster_barrier();
  if (rank == 0 && warp == 0) {
    balance = 0.0;
    if (lane < cluster) {
      uint32_t at;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(&part))), "r"(lane));
      asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(balance) : "r"(at) : "memory");
    }
    balance = warp_sum_f64(balance);
    z = warp_sum_f64(fold_z[lane]);
    n = fold_n[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    const double kept = static_cast<double>(n);
    if (lane == 0) {
      if (groups == 1) {
        write_totals(balance, z, kept, n > 0, loss, z_loss);
        table[s.experts] = n > 0 ? static_cast<float>(1.0 / kept) : 0.f;
        table[s.experts + 1] = table[s.experts];
      } else {
        in.group[group * 3] = balance;
        in.group[group * 3 + 1] = z;
        in.group[group * 3 + 2] = kept;
      }
    }
  }
  cluster_barrier();  // no CTA leaves while its part may be read
}

// The mean over the groups: one CTA.
__global__ void __launch_bounds__(kThreads)
balance_total_kernel(const double* group, int64_t groups, int experts, float* table, float* loss,
                     float* z_loss) {
  pdl_prologue();
  constexpr int WARPS = kThreads / 32;
  __shared__ double fold[4][WARPS];
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  for (int64_t g = threadIdx.x; g < groups; g += kThreads) {
    v[0] += group[g * 3];
    v[1] += group[g * 3 + 1];
    v[2] += group[g * 3 + 2];
    v[3] += group[g * 3 + 2] > 0 ? 1.0 : 0.0;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = warp_sum_f64(v[k]);
    if ((threadIdx.x & 31) == 0) fold[k][threadIdx.x >> 5] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = 0.0;
    for (int w = 0; w < WARPS; ++w) v[k] += fold[k][w];
  }
  float* scale = table + groups * experts;
  for (int64_t g = threadIdx.x; g < groups; g += kThreads) {
    const double n = group[g * 3 + 2];
    scale[g] = n > 0 ? static_cast<float>(1.0 / (v[3] * n)) : 0.f;
  }
  if (threadIdx.x == 0) {
    write_totals(v[0], v[1], v[2], static_cast<int>(v[3]), loss, z_loss);
    scale[groups] = v[2] > 0 ? static_cast<float>(1.0 / v[2]) : 0.f;
  }
}

// grad_logits; rows that the mask leaves out get zeros.
template <typename T, bool VEC, int LPT, int WPL, int U>
__global__ void __launch_bounds__(kThreads, 2)
balance_backward_kernel(const T* logits, const uint8_t* mask, const float2* stats, const float* table, const float* grad_loss, const float* grad_z,
                        T* grad, const Shape s, int64_t ldo) {
  using L = Load<T, VEC>;
  constexpr int N = L::N;
  constexpr int TOKENS = 32 / LPT;
  constexpr int WARPS = kThreads / 32;
  pdl_prologue();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lane_in_token = lane % LPT;
  const int64_t group = blockIdx.y, base = group * s.tokens;
  const int tokens = static_cast<int>(s.tokens);
  logits += base * s.ld;
  grad += base * ldo;
  stats += base;
  if (mask != nullptr) mask += base;
  const float* scale = table + static_cast<int64_t>(gridDim.y) * s.experts;
  const float by_balance = grad_loss == nullptr ? 0.f : *grad_loss * scale[group];
  const float by_z = grad_z == nullptr ? 0.f : 2.f * *grad_z * scale[gridDim.y];
  float f[WPL][N];
#pragma unroll
  for (int i = 0; i < WPL; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = (lane_in_token + i * LPT) * N + j;
      f[i][j] = e < s.experts ? table[group * s.experts + e] : 0.f;
    }
  constexpr int TILE = WARPS * TOKENS * U;
  // which of the next tile's tokens count: a tile ahead, so that the logits do not wait for the mask
  bool kept_next[U];
  auto look = [&](int64_t tile) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = tile * TILE + (warp * U + u) * TOKENS + lane / LPT;
      kept_next[u] = t < tokens && (mask == nullptr || mask[t] != 0);
    }
  };
  // loads behind the last expert are never made and stay -inf; those of a token that does not count are stale and not used
  typename L::Raw raw[U][WPL];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < WPL; ++i) raw[u][i] = L::lowest();
  look(blockIdx.x);
  for (int64_t tile = blockIdx.x; tile * TILE < tokens; tile += s.chunks) {
    const int t0 = static_cast<int>(tile) * TILE + warp * TOKENS * U;
    float2 stat[U];
    bool keep[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * TOKENS + lane / LPT;
      keep[u] = kept_next[u];
      stat[u] = keep[u] ? stats[t] : make_float2(0.f, 1.f);
#pragma unroll
      for (int i = 0; i < WPL; ++i) {
        const int e = (lane_in_token + i * LPT) * N;
        if (keep[u] && e < s.experts) raw[u][i] = L::get(logits + t * s.ld + e);
      }
    }
    look(tile + s.chunks);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * TOKENS + lane / LPT;
      float p[WPL][N];
      const float inv = __frcp_rn(stat[u].y);
      float inner = 0.f;
#pragma unroll
      for (int i = 0; i < WPL; ++i) {
        L::unpack(raw[u][i], p[i]);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          p[i][j] = exp_from(p[i][j], stat[u].x) * inv;
          inner = fmaf(p[i][j], f[i][j], inner);
        }
      }
      inner = lanes_sum<LPT>(inner);
      const float shift = by_z * (stat[u].x + logf(stat[u].y)) - by_balance * inner;
#pragma unroll
      for (int i = 0; i < WPL; ++i) {
        const int e = (lane_in_token + i * LPT) * N;
        if (t >= tokens || e >= s.experts) continue;
#pragma unroll
        for (int j = 0; j < N; ++j) p[i][j] = keep[u] ? p[i][j] * fmaf(by_balance, f[i][j], shift) : 0.f;
        L::put(grad + t * ldo + e, p[i]);
      }
    }
  }
}

// CTAs of a group, each with a line of sums: as many as run at once over all groups.  (Three times as many, so that the CTAs
// of short sequences leave their room to others, gained nothing: [32, 4001, 256] fp32 forward 45 us against 43.)
int chunks_for(int64_t groups, int64_t tokens) {
  const int64_t fill = std::max<int64_t>(1, static_cast<int64_t>(sm_count()) * 2 / std::max<int64_t>(groups, 1));
  return static_cast<int>(std::min(fill, std::max<int64_t>(1, ceil_div(tokens, 32))));
}

size_t scratch_layout(int64_t groups, int64_t chunks, int64_t experts, char* base, Partials* out) {
  const size_t lines = static_cast<size_t>(groups) * static_cast<size_t>(chunks);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 15) / 16 * 16;
    return base + here;
  };
  Partials p;
  p.group = reinterpret_cast<double*>(take(static_cast<size_t>(groups) * 3 * sizeof(double)));
  p.probs = reinterpret_cast<float*>(take(lines * experts * sizeof(float)));
  p.picks = reinterpret_cast<int*>(take(lines * experts * sizeof(int)));
  p.z = reinterpret_cast<float*>(take(lines * sizeof(float)));
  p.kept = reinterpret_cast<int*>(take(lines * sizeof(int)));
  if (out != nullptr) *out = p;
  return at;
}

// Lanes per token, loads per lane and tokens at a time: eight loads in flight.  Rows in words take eight lanes (128 bytes of
// a row at a time) until a lane would hold more than 32 values of a row; rows element by element take a warp.
template <typename T, bool VEC, typename F>
int with_lanes(int experts, F&& call) {
  constexpr int N = Load<T, VEC>::N;
#define B200_LANES(LPT, WPL, U) return call(std::integral_constant<int, LPT>(), std::integral_constant<int, WPL>(), std::integral_constant<int, U>())
  const int loads = static_cast<int>(ceil_div(experts, N));
  if constexpr (N == 1) {
    if (loads <= 8) B200_LANES(8, 1, 4);
    if (loads <= 32) B200_LANES(32, 1, 8);
    if (loads <= 64) B200_LANES(32, 2, 8);
    if (loads <= 128) B200_LANES(32, 4, 8);
    if (loads <= 256) B200_LANES(32, 8, 4);
    if (loads <= 512) B200_LANES(32, 16, 2);
    B200_LANES(32, 32, 1);
  } else {
    constexpr int W = 32 / N;  // loads of a row that a lane may hold
    if (loads <= 1) B200_LANES(1, 1, 4);
    if (loads <= 2) B200_LANES(2, 1, 4);
    if (loads <= 4) B200_LANES(4, 1, 4);
    if (loads <= 8) B200_LANES(8, 1, 8);
    if (loads <= 16) B200_LANES(8, 2, 4);
    if (loads <= 32) B200_LANES(8, 4, 2);
    if (loads <= 64) B200_LANES(64 / W, W, 8 / W);
    if (N == 8 || loads <= 128) B200_LANES(128 / W, W, 8 / W);
    B200_LANES(32, W, 8 / W);  // fp32 only: 256 words
  }
#undef B200_LANES
}

template <typename... Params, typename... Args>
void launch_cluster(void (*kernel)(Params...), unsigned grid, unsigned block, unsigned cluster, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = block;
  config.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = pdl_enabled() ? 2 : 1;
  (void)cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
}

int check_shape(const char* fn, int64_t groups, int64_t tokens, int64_t experts, int64_t top_k, int dtype) {
  if (!dtype_ok(dtype)) return fail(B200_ERR_DTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (groups < 0 || tokens < 0) return fail(B200_ERR_SHAPE, "%s: negative size", fn);
  if (groups > 65535) return fail(B200_ERR_SHAPE, "%s: groups=%lld exceeds 65535", fn, (long long)groups);
  if (tokens > (1LL << 30)) return fail(B200_ERR_SHAPE, "%s: more than 2^30 tokens", fn);
  if (experts < 1 || experts > kMaxExperts) return fail(B200_ERR_SHAPE, "%s: experts=%lld is not in 1..%d", fn, (long long)experts, kMaxExperts);
  if (top_k < 1 || top_k > kMaxTopK || top_k > experts) return fail(B200_ERR_SHAPE, "%s: top_k=%lld is not in 1..min(experts, %d)", fn, (long long)top_k, kMaxTopK);
  if (groups * tokens * top_k > (1LL << 30)) return fail(B200_ERR_SHAPE, "%s: more than 2^30 picks", fn);
  return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_moe_balance_scratch_bytes(int64_t groups, int64_t tokens, int64_t experts, size_t* bytes) {
  B200_REQUIRE_PTR(bytes);
  if (int rc = check_shape(__func__, groups, tokens, experts, 1, B200_F32)) return rc;
  if (int rc = check_device()) return rc;
  *bytes = scratch_layout(groups, chunks_for(groups, tokens), experts, nullptr, nullptr);
  return B200_OK;
}

extern "C" int b200_moe_balance_loss(const void* logits, const int32_t* indices, const uint8_t* mask, float* balance, float* z, int32_t* counts,
                                     float* stats, float* table, int64_t groups, int64_t tokens, int64_t experts, int64_t top_k,
                                     int64_t ld_logits, int logits_dtype, void* scratch, size_t scratch_bytes, void* stream) {
  if (int rc = check_shape(__func__, groups, tokens, experts, top_k, logits_dtype)) return rc;
  B200_REQUIRE_PTR(balance);
  B200_REQUIRE_PTR(z);
  B200_REQUIRE_PTR(table);
  if (groups > 0) {
    B200_REQUIRE_PTR(counts);
    B200_REQUIRE_PTR(scratch);
  }
  if (groups > 0 && tokens > 0) {
    B200_REQUIRE_PTR(logits);
    B200_REQUIRE_PTR(indices);
  }
  if (ld_logits < experts) return fail(B200_ERR_SHAPE, "%s: leading dimension smaller than experts", __func__);
  const size_t es = dtype_size(logits_dtype);
  if (!aligned(logits, es) || !aligned(indices, 4) || !aligned(stats, 8) || !aligned(table, 4) || !aligned(counts, 4))
    return fail(B200_ERR_ALIGNMENT, "%s: pointer not aligned to its element size (stats: 8 bytes)", __func__);
  if (int rc = check_device()) return rc;
  Shape s;
  s.tokens = tokens, s.ld = ld_logits, s.experts = static_cast<int>(experts), s.top_k = static_cast<int>(top_k), s.chunks = chunks_for(groups, tokens);
  Partials part;
  const size_t need = scratch_layout(groups, s.chunks, experts, static_cast<char*>(scratch), &part);
  if (scratch_bytes < need || !aligned(scratch, 16))
    return fail(B200_ERR_SCRATCH, "%s: scratch needs %zu bytes, 16-byte aligned (got %zu)", __func__, need, scratch_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = B200_OK;
  if (groups > 0) {
    const dim3 grid(static_cast<unsigned>(s.chunks), static_cast<unsigned>(groups));
    B200_DISPATCH_DTYPE(logits_dtype, T, {
      const T* l = static_cast<const T*>(logits);
      float2* saved = reinterpret_cast<float2*>(stats);
      const bool vec = experts % Num<T>::kVec == 0 && ld_logits % Num<T>::kVec == 0 && aligned(logits, 16);
      if (vec)
        rc = with_lanes<T, true>(s.experts, [&](auto lanes, auto loads, auto at_a_time) {
          launch(balance_sums_kernel<T, true, lanes.value, loads.value, at_a_time.value>, grid, kThreads, 0, st, l, indices, mask, saved, s, part);
          return after_launch("balance_sums_kernel");
        });
      else
        rc = with_lanes<T, false>(s.experts, [&](auto lanes, auto loads, auto at_a_time) {
          launch(balance_sums_kernel<T, false, lanes.value, loads.value, at_a_time.value>, grid, kThreads, 0, st, l, indices, mask, saved, s, part);
          return after_launch("balance_sums_kernel");
        });
    });
    if (rc) return rc;
    const int cluster = static_cast<int>(std::min<int64_t>(kMaxCluster, ceil_div(experts, 32)));
    launch_cluster(balance_group_kernel, static_cast<unsigned>(groups * cluster), kGroupThreads, static_cast<unsigned>(cluster), st, s, part,
                   static_cast<int>(groups), cluster, counts, table, balance, z);
    if ((rc = after_launch("balance_group_kernel"))) return rc;
  }
  if (groups != 1) {
    launch(balance_total_kernel, 1, kThreads, 0, st, static_cast<const double*>(part.group), groups, s.experts, table, balance, z);
    if ((rc = after_launch("balance_total_kernel"))) return rc;
  }
  return B200_OK;
}

extern "C" int b200_moe_balance_loss_backward(const void* logits, const uint8_t* mask, const float* stats, const float* table,
                                              const float* grad_balance, const float* grad_z, void* grad_logits, int64_t groups, int64_t tokens,
                                              int64_t experts, int64_t ld_logits, int64_t ld_grad, int logits_dtype, void* stream) {
  if (int rc = check_shape(__func__, groups, tokens, experts, 1, logits_dtype)) return rc;
  if (groups == 0 || tokens == 0) return B200_OK;
  B200_REQUIRE_PTR(logits);
  B200_REQUIRE_PTR(stats);
  B200_REQUIRE_PTR(table);
  B200_REQUIRE_PTR(grad_logits);
  if (ld_logits < experts || ld_grad < experts) return fail(B200_ERR_SHAPE, "%s: leading dimension smaller than experts", __func__);
  const size_t es = dtype_size(logits_dtype);
  if (!aligned(logits, es) || !aligned(grad_logits, es) || !aligned(stats, 8) || !aligned(table, 4) || !aligned(grad_balance, 4) || !aligned(grad_z, 4))
    return fail(B200_ERR_ALIGNMENT, "%s: pointer not aligned to its element size (stats: 8 bytes)", __func__);
  if (int rc = check_device()) return rc;
  Shape s;
  s.tokens = tokens, s.ld = ld_logits, s.experts = static_cast<int>(experts), s.top_k = 1, s.chunks = chunks_for(groups, tokens);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(s.chunks), static_cast<unsigned>(groups));
  int rc = B200_OK;
  B200_DISPATCH_DTYPE(logits_dtype, T, {
    const T* l = static_cast<const T*>(logits);
    T* out = static_cast<T*>(grad_logits);
    const float2* saved = reinterpret_cast<const float2*>(stats);
    const bool vec = experts % Num<T>::kVec == 0 && ld_logits % Num<T>::kVec == 0 && ld_grad % Num<T>::kVec == 0 && aligned(logits, 16) && aligned(grad_logits, 16);
    if (vec)
      rc = with_lanes<T, true>(s.experts, [&](auto lanes, auto loads, auto at_a_time) {
        launch(balance_backward_kernel<T, true, lanes.value, loads.value, at_a_time.value>, grid, kThreads, 0, st, l, mask, saved, table, grad_balance, grad_z, out, s, ld_grad);
        return after_launch("balance_backward_kernel");
      });
    else
      rc = with_lanes<T, false>(s.experts, [&](auto lanes, auto loads, auto at_a_time) {
        launch(balance_backward_kernel<T, false, lanes.value, loads.value, at_a_time.value>, grid, kThreads, 0, st, l, mask, saved, table, grad_balance, grad_z, out, s, ld_grad);
        return after_launch("balance_backward_kernel");
      });
  });
  return rc;
}
