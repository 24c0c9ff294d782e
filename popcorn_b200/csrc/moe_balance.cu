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
// leaves one line of sums, a second small kernel adds the lines up in a fixed order in fp64.  Backward: the logits read
// again, the gradient written; row maximum and sum come from the forward pass (8 bytes a token).
#include <algorithm>

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
  static __device__ __forceinline__ void get(const T* p, float (&f)[N]) { Num<T>::unpack(ld_stream(p), f); }
  static __device__ __forceinline__ void put(T* p, const float (&f)[N]) { st_stream(p, Num<T>::pack(f)); }
};
template <typename T>
struct Load<T, false> {
  static constexpr int N = 1;
  static __device__ __forceinline__ void get(const T* p, float (&f)[1]) { f[0] = Num<T>::up(*p); }
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

__device__ __forceinline__ int64_t chunk_start(const Shape& s, int chunk) { return s.tokens * chunk / s.chunks; }

template <typename T, bool VEC, int LPT, int WPL>
__global__ void __launch_bounds__(kThreads)
balance_sums_kernel(const T* logits, const int32_t* indices, const uint8_t* mask,
                    float2* stats, const Shape s, const Partials out) {
  using L = Load<T, VEC>;
  constexpr int N = L::N;
  constexpr int TOKENS = 32 / LPT;  // tokens of a warp at a time
  constexpr int WARPS = kThreads / 32;
  pdl_prologue();
  __shared__ int picks[kMaxExperts];
  __shared__ float fold[WARPS][LPT * WPL * N];
  __shared__ float fold_z[WARPS];
  __shared__ int fold_n[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lane_in_token = lane % LPT;
  const int64_t group = blockIdx.y, base = group * s.tokens;
  const int64_t first = chunk_start(s, blockIdx.x), last = chunk_start(s, blockIdx.x + 1);
  for (int e = threadIdx.x; e < s.experts; e += kThreads) picks[e] = 0;
  __syncthreads();
  float sums[WPL][N], z = 0.f;
  int kept = 0;
#pragma unroll
  for (int i = 0; i < WPL; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) sums[i][j] = 0.f;
  // every lane of a warp runs the same number of iterations: the shuffles need them all
  for (int64_t t0 = first + warp * TOKENS; t0 < last; t0 += WARPS * TOKENS) {
    const int64_t t = t0 + lane / LPT;
    const bool keep = t < last && (mask == nullptr || mask[base + t] != 0);
    float v[WPL][N], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < WPL; ++i) {
      const int e = (lane_in_token + i * LPT) * N;
#pragma unroll
      for (int j = 0; j < N; ++j) v[i][j] = -INFINITY;
      if (keep && e < s.experts) L::get(logits + (base + t) * s.ld + e, v[i]);
#pragma unroll
      for (int j = 0; j < N; ++j) top = fmaxf(top, v[i][j]);
    }
    top = lanes_max<LPT>(top);
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < WPL; ++i) {
      const bool there = (lane_in_token + i * LPT) * N < s.experts;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        v[i][j] = there ? expf(v[i][j] - top) : 0.f;  // a row of -inf alone is NaN, as in a softmax
        total += v[i][j];
      }
    }
    total = lanes_sum<LPT>(total);
    if (keep) {
      const float inv = __frcp_rn(total);
#pragma unroll
      for (int i = 0; i < WPL; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) sums[i][j] = fmaf(v[i][j], inv, sums[i][j]);
      if (lane_in_token == 0) {
        const float lse = top + logf(total);
        z = fmaf(lse, lse, z);
        ++kept;
        if (stats != nullptr) stats[base + t] = make_float2(top, total);
      }
    }
  }
  for (int64_t i = first * s.top_k + threadIdx.x; i < last * s.top_k; i += kThreads) {
    if (mask != nullptr && mask[base + i / s.top_k] == 0) continue;
    const int e = indices[base * s.top_k + i];
    if (static_cast<unsigned>(e) < static_cast<unsigned>(s.experts)) atomicAdd(&picks[e], 1);  // whole numbers: any order
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
// One CTA per group adds up its lines: the 32 lanes of a warp take 32 experts, the warps every WARPS-th line.
constexpr int kGroupThreads = 1024;
__device__ void write_totals(double balance, double z, double kept, int used, float* loss, float* z_loss) {
  *loss = used > 0 ? static_cast<float>(balance / used) : 0.f;
  *z_loss = kept > 0 ? static_cast<float>(z / kept) : 0.f;
}
__global__ void __launch_bounds__(kGroupThreads)
balance_group_kernel(const Shape s, const Partials in, int groups, int32_t* counts, float* table,
                     float* loss, float* z_loss) {
  pdl_prologue();
  constexpr int WARPS = kGroupThreads / 32;
  __shared__ double fold_p[WARPS][32];
  __shared__ int fold_c[WARPS][32];
  __shared__ double fold_z[WARPS];
  __shared__ long long fold_n[WARPS];
  __shared__ double total_z;
  __shared__ long long total_n;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t group = blockIdx.x, line0 = group * s.chunks;
  double z = 0.0;
  long long n = 0;
  for (int c = threadIdx.x; c < s.chunks; c += kGroupThreads) {
    z += in.z[line0 + c];
    n += in.kept[line0 + c];
  }
  z = warp_sum_f64(z);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if (lane == 0) {
    fold_z[warp] = z;
    fold_n[warp] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    long long kept = 0;
    for (int w = 0; w < WARPS; ++w) {
      sum += fold_z[w];
      kept += fold_n[w];
    }
    total_z = sum;
    total_n = kept;
  }
  __syncthreads();
  const double kept = static_cast<double>(total_n);
  double balance = 0.0;  // of warp 0's lanes
  for (int e0 = 0; e0 < s.experts; e0 += 32) {
    const int e = e0 + lane;
    double p = 0.0;
    int picks = 0;
    if (e < s.experts) {
#pragma unroll 4
      for (int c = warp; c < s.chunks; c += WARPS) {
        p += in.probs[(line0 + c) * s.experts + e];
        picks += in.picks[(line0 + c) * s.experts + e];
      }
    }
    fold_p[warp][lane] = p;
    fold_c[warp][lane] = picks;
    __syncthreads();
    if (warp == 0 && e < s.experts) {
      p = 0.0;
      picks = 0;
      for (int w = 0; w < WARPS; ++w) {
        p += fold_p[w][lane];
        picks += fold_c[w][lane];
      }
      const double f = kept > 0 ? static_cast<double>(picks) * s.experts / (kept * s.top_k) : 0.0;
      counts[group * s.experts + e] = picks;
      table[group * s.experts + e] = static_cast<float>(f);
      if (kept > 0) balance += f * p / kept;
    }
    __syncthreads();
  }
  if (warp == 0) {
    balance = warp_sum_f64(balance);
    if (lane == 0) {
      if (groups == 1) {
        write_totals(balance, total_z, kept, kept > 0, loss, z_loss);
        table[s.experts] = kept > 0 ? static_cast<float>(1.0 / kept) : 0.f;
        table[s.experts + 1] = table[s.experts];
      } else {
        in.group[group * 3] = balance;
        in.group[group * 3 + 1] = total_z;
        in.group[group * 3 + 2] = kept;
      }
    }
  }
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
template <typename T, bool VEC, int LPT, int WPL>
__global__ void __launch_bounds__(kThreads)
balance_backward_kernel(const T* logits, const uint8_t* mask, const float2* stats,
                        const float* table, const float* grad_loss, const float* grad_z,
                        T* grad, const Shape s, int64_t ldo) {
  using L = Load<T, VEC>;
  constexpr int N = L::N;
  constexpr int TOKENS = 32 / LPT;
  constexpr int WARPS = kThreads / 32;
  pdl_prologue();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lane_in_token = lane % LPT;
  const int64_t group = blockIdx.y, base = group * s.tokens;
  const int64_t first = chunk_start(s, blockIdx.x), last = chunk_start(s, blockIdx.x + 1);
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
  for (int64_t t0 = first + warp * TOKENS; t0 < last; t0 += WARPS * TOKENS) {
    const int64_t t = t0 + lane / LPT;
    const bool live = t < last, keep = live && (mask == nullptr || mask[base + t] != 0);
    const float2 stat = keep ? stats[base + t] : make_float2(0.f, 1.f);
    const float inv = __frcp_rn(stat.y);
    float p[WPL][N], inner = 0.f;
#pragma unroll
    for (int i = 0; i < WPL; ++i) {
      const int e = (lane_in_token + i * LPT) * N;
#pragma unroll
      for (int j = 0; j < N; ++j) p[i][j] = -INFINITY;
      if (keep && e < s.experts) L::get(logits + (base + t) * s.ld + e, p[i]);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        p[i][j] = e < s.experts ? expf(p[i][j] - stat.x) * inv : 0.f;
        inner = fmaf(p[i][j], f[i][j], inner);
      }
    }
    inner = lanes_sum<LPT>(inner);
    const float shift = by_z * (stat.x + logf(stat.y)) - by_balance * inner;
#pragma unroll
    for (int i = 0; i < WPL; ++i) {
      const int e = (lane_in_token + i * LPT) * N;
      if (!live || e >= s.experts) continue;
#pragma unroll
      for (int j = 0; j < N; ++j) p[i][j] = keep ? p[i][j] * fmaf(by_balance, f[i][j], shift) : 0.f;
      L::put(grad + (base + t) * ldo + e, p[i]);
    }
  }
}

// Lines of sums of a group: as many CTAs as fill the GPU twice over all groups, each with at least 32 tokens.
int chunks_for(int64_t groups, int64_t tokens) {
  const int64_t fill = ceil_div(static_cast<int64_t>(sm_count()) * 2, std::max<int64_t>(groups, 1));
  return static_cast<int>(std::max<int64_t>(1, std::min(fill, ceil_div(tokens, 32))));
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

// Lanes per token and loads per lane for a row of `loads` loads.  A lane holds eight values of a row (a 16-bit word, two
// fp32 words) up to 256 experts, so that a row's maximum and sum need few shuffles; more for longer rows.
template <typename T, bool VEC, typename F>
int with_lanes(int experts, F&& call) {
  constexpr int N = Load<T, VEC>::N, W = 8 / N;
  const int lanes = static_cast<int>(ceil_div(experts, 8));
  if (lanes <= 1) return call(std::integral_constant<int, 1>(), std::integral_constant<int, W>());
  if (lanes <= 2) return call(std::integral_constant<int, 2>(), std::integral_constant<int, W>());
  if (lanes <= 4) return call(std::integral_constant<int, 4>(), std::integral_constant<int, W>());
  if (lanes <= 8) return call(std::integral_constant<int, 8>(), std::integral_constant<int, W>());
  if (lanes <= 16) return call(std::integral_constant<int, 16>(), std::integral_constant<int, W>());
  if (lanes <= 32) return call(std::integral_constant<int, 32>(), std::integral_constant<int, W>());
  if (lanes <= 64) return call(std::integral_constant<int, 32>(), std::integral_constant<int, 2 * W>());
  return call(std::integral_constant<int, 32>(), std::integral_constant<int, 4 * W>());
}

int check_shape(const char* fn, int64_t groups, int64_t tokens, int64_t experts, int64_t top_k, int dtype) {
  if (!dtype_ok(dtype)) return fail(B200_ERR_DTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (groups < 0 || tokens < 0) return fail(B200_ERR_SHAPE, "%s: negative size", fn);
  if (groups > 65535) return fail(B200_ERR_SHAPE, "%s: groups=%lld exceeds 65535", fn, (long long)groups);
  if (tokens > 0x7fffffffLL || groups * tokens > 0x7fffffffLL) return fail(B200_ERR_SHAPE, "%s: more than 2^31-1 tokens", fn);
  if (experts < 1 || experts > kMaxExperts) return fail(B200_ERR_SHAPE, "%s: experts=%lld is not in 1..%d", fn, (long long)experts, kMaxExperts);
  if (top_k < 1 || top_k > kMaxTopK || top_k > experts) return fail(B200_ERR_SHAPE, "%s: top_k=%lld is not in 1..min(experts, %d)", fn, (long long)top_k, kMaxTopK);
  if (groups * tokens * top_k > 0x7fffffffLL) return fail(B200_ERR_SHAPE, "%s: more than 2^31-1 picks", fn);
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
        rc = with_lanes<T, true>(s.experts, [&](auto lanes, auto loads) {
          launch(balance_sums_kernel<T, true, lanes.value, loads.value>, grid, kThreads, 0, st, l, indices, mask, saved, s, part);
          return after_launch("balance_sums_kernel");
        });
      else
        rc = with_lanes<T, false>(s.experts, [&](auto lanes, auto loads) {
          launch(balance_sums_kernel<T, false, lanes.value, loads.value>, grid, kThreads, 0, st, l, indices, mask, saved, s, part);
          return after_launch("balance_sums_kernel");
        });
    });
    if (rc) return rc;
    launch(balance_group_kernel, static_cast<unsigned>(groups), kGroupThreads, 0, st, s, part, static_cast<int>(groups), counts, table, balance, z);
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
      rc = with_lanes<T, true>(s.experts, [&](auto lanes, auto loads) {
        launch(balance_backward_kernel<T, true, lanes.value, loads.value>, grid, kThreads, 0, st, l, mask, saved, table, grad_balance, grad_z, out, s, ld_grad);
        return after_launch("balance_backward_kernel");
      });
    else
      rc = with_lanes<T, false>(s.experts, [&](auto lanes, auto loads) {
        launch(balance_backward_kernel<T, false, lanes.value, loads.value>, grid, kThreads, 0, st, l, mask, saved, table, grad_balance, grad_z, out, s, ld_grad);
        return after_launch("balance_backward_kernel");
      });
  });
  return rc;
}
