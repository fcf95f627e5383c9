// Routing of tokens to experts (gdn_route_experts):
//
//   s_e = exp(l_e - max l) / sum exp(l - max l)   or   1 / (1 + exp(-l_e))
//   c_e = s_e + bias_e;  of G equal ranges of experts, the top_groups with the largest sums of their group_best best c
//   the k largest c of those, ties to the lowest index;  w = s there, over their sum (renormalize), times scale
//
// Scores are formed in 64 bits: which of two experts is taken must not hang on how a score was rounded, and at a
// token's few hundred experts the 64-bit exponentials (full rate on gfx950) are not what the time goes to.
//
// LPT lanes share a token, lane l holding its experts l, l + LPT, ...; the k rounds of an arg max, which bound it, are
// VALU moves between lanes.  64 lanes a token finish a decode step's few tokens soonest, 32 take fewer instructions for
// many.
#include <climits>
#include <cmath>

#include "gdn_common.hpp"

namespace {

using namespace gdn;

constexpr int kMaxExperts = 1024;
constexpr int kMaxChoices = 64;
constexpr int kMaxGroups = 64;
constexpr int kThreads = 256;

struct RouteParams {
  const void* logits;
  int dt;
  int64_t ld;
  const float* bias;
  const int* n_new;
  int* indices;
  float* weights;
  int64_t N;
  int T, E, k, groups, top_groups, group_best;
  bool sigmoid, renormalize;
  double scale;
};

// The value of the lane that step s of a reduction meets: inside 16 lanes, then the other 16, then the other 32.
__device__ __forceinline__ int partner(int x, int s) {
  const bool odd = (threadIdx.x >> (s == 4 ? 4 : 5)) & 1;
  switch (s) {
    case 0: return __builtin_amdgcn_mov_dpp(x, GDN_DPP_QUAD_XOR1, 0xF, 0xF, false);
    case 1: return __builtin_amdgcn_mov_dpp(x, GDN_DPP_QUAD_XOR2, 0xF, 0xF, false);
    case 2: return __builtin_amdgcn_mov_dpp(x, GDN_DPP_HALF_MIRROR, 0xF, 0xF, false);
    case 3: return __builtin_amdgcn_mov_dpp(x, GDN_DPP_ROW_MIRROR, 0xF, 0xF, false);
    case 4: {  // [0]: the even rows in both places, [1]: the odd ones
      const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
      return odd ? r[0] : r[1];
    }
    default: {
      const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
      return odd ? r[0] : r[1];
    }
  }
}
__device__ __forceinline__ double partner(double x, int s) {
  const int64_t b = __builtin_bit_cast(int64_t, x);
  const uint32_t lo = partner(static_cast<int>(b), s), hi = partner(static_cast<int>(b >> 32), s);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

template <int LPT, class F, class X>
__device__ __forceinline__ X over_lanes(X x, F f) {
#pragma unroll
  for (int s = 0; s < (LPT == 64 ? 6 : LPT == 32 ? 5 : 4); ++s) x = f(x, partner(x, s));
  return x;
}
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }  // (of a number and NaN the number)
__device__ __forceinline__ double added(double a, double b) { return a + b; }
__device__ __forceinline__ int smaller(int a, int b) { return a < b ? a : b; }

template <int LPT, int VPL>
__global__ __launch_bounds__(kThreads) void route_kernel(const RouteParams p) {
  constexpr int TPB = kThreads / LPT;  // tokens
  // the experts' c where groups are scored, then the groups' and who stays
  __shared__ double group_c[kThreads * VPL];
  __shared__ double group_s[TPB * kMaxGroups];
  const int lane = threadIdx.x % LPT, slot = threadIdx.x / LPT;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * TPB + slot;
  const int64_t row = n < p.N ? n : p.N - 1;  // (every lane stays, for the barriers)
  const bool real = !p.n_new || static_cast<int>(row % p.T) < p.n_new[row / p.T];

  double c[VPL];  // logits, then scores, then what the choice goes by
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const int e = lane + v * LPT;
    c[v] = e < p.E ? static_cast<double>(load_any(p.logits, p.dt, row * p.ld + e)) : -INFINITY;
  }
  double top = 0.0, sum = 1.0;
  if (!p.sigmoid) {
    top = -INFINITY;
#pragma unroll
    for (int v = 0; v < VPL; ++v) top = larger(top, c[v]);
    top = over_lanes<LPT>(top, larger);
    if (top == -INFINITY) top = 0.0;  // nothing but -inf (and NaN): scores of 0
    sum = 0.0;
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if (lane + v * LPT < p.E) sum += exp(c[v] - top);
    sum = over_lanes<LPT>(sum, added);
    if (sum == 0.0) sum = 1.0;
  }
  auto score = [&](double x) { return p.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - top) / sum; };
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const int e = lane + v * LPT;
    c[v] = score(c[v]);
    if (p.bias && e < p.E) c[v] += static_cast<double>(p.bias[e]);
    if (p.top_groups < p.groups && e < p.E) group_c[slot * (LPT * VPL) + e] = c[v];
  }
  uint32_t left = 0;  // which of the lane's experts can be chosen
#pragma unroll
  for (int v = 0; v < VPL; ++v) left |= (lane + v * LPT < p.E ? 1u : 0u) << v;

  if (p.top_groups < p.groups) {
    const int width = p.E / p.groups;
    double* mine = group_s + slot * kMaxGroups;
    __syncthreads();
    for (int g = lane; g < p.groups; g += LPT) {
      const double* at = group_c + slot * (LPT * VPL) + g * width;
      double best = -INFINITY, second = -INFINITY;
      for (int i = 0; i < width; ++i) {  // (NaN counts as -inf)
        const double x = larger(at[i], -INFINITY);
        second = larger(second, x < best ? x : best);
        best = larger(best, x);
      }
      // (+inf and -inf, of biases, have no sum: NaN, which would stand before no other group and behind none)
      mine[g] = p.group_best > 1 && width > 1 ? larger(best + second, -INFINITY) : best;
    }
    __syncthreads();
    uint64_t stay = 0;  // a lane's groups that stay, then all lanes'
    for (int g = lane; g < p.groups; g += LPT) {
      const double s = mine[g];
      int before = 0;  // groups that come first: larger, or as large with a lower index
      for (int o = 0; o < p.groups; ++o) before += mine[o] > s || (mine[o] == s && o < g) ? 1 : 0;
      stay |= static_cast<uint64_t>(before < p.top_groups) << g;
    }
    const uint32_t lo = over_lanes<LPT>(static_cast<int>(stay), [](int a, int b) { return a | b; });
    const uint32_t hi = over_lanes<LPT>(static_cast<int>(stay >> 32), [](int a, int b) { return a | b; });
    stay = static_cast<uint64_t>(hi) << 32 | lo;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int e = lane + v * LPT;
      if (e < p.E && !(stay >> (e / width) & 1)) left &= ~(1u << v);
    }
  }

  // k times the largest c that is left (NaN counts below every number), the lowest index of equals; choice j is lane j's
  int chosen = -1;
  double w = 0.0;
#pragma unroll
  for (int v = 0; v < VPL; ++v)
    if (!(left >> v & 1)) c[v] = -INFINITY;
  for (int j = 0; j < p.k; ++j) {
    double best = -INFINITY;
#pragma unroll
    for (int v = 0; v < VPL; ++v) best = larger(best, c[v]);
    best = over_lanes<LPT>(best, larger);
    int at = INT_MAX;
    // (what cannot be chosen, or has been, is -inf, which only the last ones left may be too)
    const uint32_t open = best > -INFINITY ? ~0u : left;
#pragma unroll
    for (int v = VPL - 1; v >= 0; --v)
      if (c[v] == best && open >> v & 1) at = lane + v * LPT;
    at = over_lanes<LPT>(at, smaller);
    if (at == INT_MAX) {  // nothing but NaN is left
#pragma unroll
      for (int v = VPL - 1; v >= 0; --v)
        if (left >> v & 1) at = lane + v * LPT;
      at = over_lanes<LPT>(at, smaller);
      best = NAN;
    }
    if (lane == j) {  // (k <= LPT)
      chosen = at;
      w = best;
    }
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      if (at != lane + v * LPT) continue;
      c[v] = -INFINITY;
      left &= ~(1u << v);
    }
  }
  if (lane >= p.k) w = 0.0;
  else if (p.bias) w = score(static_cast<double>(load_any(p.logits, p.dt, row * p.ld + chosen)));
  if (p.renormalize) {
    const double all = over_lanes<LPT>(w, added);
    w = all == 0.0 ? 0.0 : w / all;
  }
  if (n < p.N && lane < p.k) {
    p.indices[n * p.k + lane] = real ? chosen : -1;
    p.weights[n * p.k + lane] = real ? static_cast<float>(w * p.scale) : 0.0f;
  }
}

template <int LPT, int VPL>
void launch(const RouteParams& p, hipStream_t st) {
  const int64_t blocks = (p.N + kThreads / LPT - 1) / (kThreads / LPT);
  hipLaunchKernelGGL((route_kernel<LPT, VPL>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, p);
}

}  // namespace

extern "C" int gdn_route_experts(const void* logits, int dtype, int64_t ld, const float* bias, const int32_t* n_new,
                                 int32_t* indices, float* weights, int64_t B, int64_t T, int64_t E, int64_t k,
                                 int sigmoid, int64_t groups, int64_t top_groups, int64_t group_best, int renormalize,
                                 double scale, void* stream) {
  using gdn_host::fail;
  if (B < 0 || T < 0 || E < 1 || E > kMaxExperts || k < 1 || k > kMaxChoices)
    return fail(GDN_ERR_INVALID, "gdn_route_experts: bad sizes B=%lld T=%lld E=%lld k=%lld (E up to %d, k up to %d)",
                (long long)B, (long long)T, (long long)E, (long long)k, kMaxExperts, kMaxChoices);
  if (groups < 1 || groups > kMaxGroups || E % groups || top_groups < 1 || top_groups > groups || group_best < 1 ||
      group_best > 2 || k > E / groups * top_groups)
    return fail(GDN_ERR_INVALID,
                "gdn_route_experts: %lld of %lld groups of %lld experts (equal groups, up to %d) cannot give %lld choices",
                (long long)top_groups, (long long)groups, (long long)E, kMaxGroups, (long long)k);
  if (!gdn_host::dtype_ok(dtype)) return fail(GDN_ERR_INVALID, "gdn_route_experts: unknown dtype");
  if (B == 0 || T == 0) return GDN_OK;
  if (T > INT32_MAX || B > INT32_MAX / T) return fail(GDN_ERR_UNSUPPORTED, "gdn_route_experts: too many tokens");
  if (!logits || !indices || !weights) return fail(GDN_ERR_INVALID, "gdn_route_experts: null pointer");
  if (ld < E) return fail(GDN_ERR_INVALID, "gdn_route_experts: rows overlap");
  if (!gdn_host::aligned(logits, dtype == GDN_DTYPE_F32 ? 4 : 2) || !gdn_host::aligned(bias, 4) ||
      !gdn_host::aligned(n_new, 4) || !gdn_host::aligned(indices, 4) || !gdn_host::aligned(weights, 4))
    return fail(GDN_ERR_INVALID, "gdn_route_experts: misaligned pointer");
  RouteParams p = {};
  p.logits = logits;
  p.dt = dtype;
  p.ld = ld;
  p.bias = bias;
  p.n_new = n_new;
  p.indices = indices;
  p.weights = weights;
  p.N = B * T;
  p.T = static_cast<int>(T);
  p.E = static_cast<int>(E);
  p.k = static_cast<int>(k);
  p.groups = static_cast<int>(groups);
  p.top_groups = static_cast<int>(top_groups);
  p.group_best = static_cast<int>(group_best);
  p.sigmoid = sigmoid != 0;
  p.renormalize = renormalize != 0;
  p.scale = scale;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  // us with 64 and 32 lanes a token, 8 of 256: 1024 tokens 6.7, 8.9; 4096 12.7, 11.2; 16384 37.6, 29.4 (16 lanes: 14.0,
  // 14.5, 28.4)
  if (p.N >= 3500 && k <= 32 && E <= 256) {
    if (E <= 64) launch<32, 2>(p, st);
    else launch<32, 8>(p, st);
  } else if (E <= 64) {
    launch<64, 1>(p, st);
  } else if (E <= 128) {
    launch<64, 2>(p, st);
  } else if (E <= 256) {
    launch<64, 4>(p, st);
  } else if (E <= 512) {
    launch<64, 8>(p, st);
  } else {
    launch<64, 16>(p, st);
  }
  return gdn_host::check_launch("gdn_route_experts");
}
