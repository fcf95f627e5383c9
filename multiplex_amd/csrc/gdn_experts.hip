// The experts of a sparse MLP (gdn_expert_mlp):
//
//   out_t = base_t + sum_j w_tj (silu(x_t G_e^T) * (x_t U_e^T)) D_e^T,  e = indices[t][j]
//
// Tokens choose k of E experts each, so an expert's products have as many rows as tokens chose it, which only the device
// knows.  The pairs (token, choice) are put in the experts' order (plan_place_kernel), every expert's cut into tiles of
// rows, and one launch runs all tiles of all experts: a workgroup finds its expert, rows and columns in the plan.  The
// launch has as many workgroups as the pairs can need at most; those past the plan's end leave.
// SwiGLU happens in the first product's epilogue (a wave forms a column of the gate and the same column of up), its
// result is rounded to bf16 as the second product's operand: the matrix units multiply bf16, and a second product of what
// the rounding leaves would double theirs.  The k results of a token wait in 20 bits a column and are summed in fp32 in the
// order of its choices: a result does not depend on where a pair came to lie in the plan.
#include <cmath>

#include "gdn_dot.hpp"

namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxChoices = 64;
// The second product's rows, the inner values, are 32-bit byte offsets from a tile's first one of up to 256, below 2 GiB.
constexpr int64_t kMostInner = (int64_t{1} << 30) / 256;

// -------------------------------------------------------------------- plan
//
// The pairs p = t k + j whose expert is one of the E, in the experts' order (from: their tokens, to: the pairs), and
// the experts' tiles of up to `rows` rows.  A chunk of the pairs is one workgroup's; with several chunks a launch
// before counts each chunk's pairs by expert, so that a workgroup knows what lies in front of its own.  Where a pair
// lies among its expert's goes by the atomics' order, which no result depends on.
constexpr int kPlanThreads = 1024;
// Pairs of a thread and of a workgroup: 2048 pairs a chunk, but up to 4096 in one (2331 pairs 2 + 5 us in two launches,
// 5.5 in one).
constexpr int kChunk = 2 * kPlanThreads, kOneChunk = 2 * kChunk;

struct PlanParams {
  const int* indices;
  int P, k, E, rows, chunks;
  int* counts;  // [chunks][E]
  TileOf* tiles;
  int* n_tiles;
  int* from;
  int* to;
};

// The chunk's pairs by expert; each of the thread's pairs' expert (-1: none) and number among its chunk's.
template <int EACH>
__device__ __forceinline__ void count_pairs(const PlanParams& p, int* hist, int (&expert)[EACH], int (&number)[EACH]) {
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int i = blockIdx.x * (EACH * kPlanThreads) + j * kPlanThreads + threadIdx.x;
    const int e = i < p.P ? p.indices[i] : -1;
    expert[j] = e < p.E ? e : -1;
  }
  for (int e = threadIdx.x; e < p.E; e += kPlanThreads) hist[e] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < EACH; ++j) number[j] = expert[j] >= 0 ? atomicAdd(&hist[expert[j]], 1) : 0;
  __syncthreads();
}

__global__ __launch_bounds__(kPlanThreads) void plan_count_kernel(const PlanParams p) {
  __shared__ int hist[kMaxExperts];
  int expert[kChunk / kPlanThreads], number[kChunk / kPlanThreads];
  count_pairs(p, hist, expert, number);
  for (int e = threadIdx.x; e < p.E; e += kPlanThreads) p.counts[blockIdx.x * p.E + e] = hist[e];
}

// Sums of x over the threads before this one, and over all.
__device__ __forceinline__ int block_before(int x, int* waves, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(s, d, 64);
    if (lane >= d) s += y;
  }
  __syncthreads();  // (waves may still be read from the last sum)
  if (lane == 63) waves[wave] = s;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    if (i < wave) before += waves[i];
    sum += waves[i];
  }
  *all = sum;
  return before + s - x;
}

template <int EACH>
__global__ __launch_bounds__(kPlanThreads) void plan_place_kernel(const PlanParams p) {
  __shared__ int hist[kMaxExperts];
  __shared__ int waves[kPlanThreads / 64];
  static_assert(kMaxExperts <= kPlanThreads, "a thread an expert");
  const int e = threadIdx.x;
  int expert[EACH], number[EACH];
  count_pairs(p, hist, expert, number);
  int mine = 0, total = 0;  // pairs of expert e in the chunks before, and in all
  if (e < p.E) {
    if (p.chunks == 1) total = hist[e];
#pragma unroll 8
    for (int c = 0; c < (p.chunks == 1 ? 0 : p.chunks); ++c) {
      const int n = p.counts[c * p.E + e];
      total += n;
      mine += c < static_cast<int>(blockIdx.x) ? n : 0;
    }
  }
  int all;
  const int first = block_before(total, waves, &all);
  const int tiles = (total + p.rows - 1) / p.rows;
  const int tile0 = block_before(tiles, waves, &all);
  if (e < p.E) hist[e] = first + mine;
  if (blockIdx.x == 0) {
    for (int i = 0; i < tiles; ++i)
      p.tiles[tile0 + i] = TileOf{e, first + i * p.rows, min(p.rows, total - i * p.rows), 0};
    if (e == 0) p.n_tiles[0] = all;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    if (expert[j] < 0) continue;
    const int i = blockIdx.x * (EACH * kPlanThreads) + j * kPlanThreads + threadIdx.x, at = hist[expert[j]] + number[j];
    p.from[at] = i / p.k;
    p.to[at] = i;
  }
}

// ------------------------------------------------------------------- combine

struct CombineParams {
  const uint16_t* y;        // [N k][H], the sums' upper halves
  const uint32_t* nibbles;  // [N k][H / 8], their next four bits
  const int* indices;
  const float* weights;
  const uint16_t* base;
  int64_t ldb;
  uint16_t* out;
  int64_t ldo;
  int64_t N;
  int H, k, E;
};

// out_t = base_t + sum_j w_tj y_tj, eight columns a thread.  Bound by reading y.
__global__ __launch_bounds__(256) void combine_kernel(const CombineParams p) {
  const int per = p.H / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t t = i / per;
  if (t >= p.N) return;
  const int c = static_cast<int>(i % per) * 8;
  float sum[CPL] = {};
  if (p.base) unpack8<GDN_DTYPE_BF16>(load_raw8<GDN_DTYPE_BF16>(p.base, t * p.ldb + c), sum);
  for (int j0 = 0; j0 < p.k; j0 += 4) {  // four rows on their way at a time (those of no expert hold anything)
    u32x4 q[4];
    uint32_t q4[4];
    float w[4];
    bool in[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int64_t j = t * p.k + min(j0 + m, p.k - 1);
      const int e = p.indices[j];
      in[m] = j0 + m < p.k && e >= 0 && e < p.E;
      w[m] = p.weights[j];
      q[m] = *reinterpret_cast<const u32x4*>(p.y + j * p.H + c);
      q4[m] = p.nibbles[(j * p.H + c) / 8];
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (!in[m]) continue;
      const f32x4 y[2] = {joined4(q[m][0], q[m][1], q4[m] << 4 & 0xf0f0f0f0u), joined4(q[m][2], q[m][3], q4[m] & 0xf0f0f0f0u)};
#pragma unroll
      for (int i = 0; i < CPL; ++i) sum[i] += w[m] * y[i / 4][i % 4];
    }
  }
  store8<GDN_DTYPE_BF16>(p.out, t * p.ldo + c, sum);
}

// ---------------------------------------------------------------- few pairs
//
// For few pairs no plan is made: as many workgroups as read each pair's weights once, the second product's waves a
// token's k experts one after the other, so that their sum needs no launch of its own.

struct FewParams {
  const uint16_t* x;
  int64_t ldx;
  const uint16_t* gate_up;
  const uint16_t* down;
  uint16_t* act;  // [N k][I]
  CombineParams c;
  int I;
};

__global__ __launch_bounds__(256) void few_up_kernel(const FewParams p) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c0 = (blockIdx.x * 4 + wave) * 2, pair = blockIdx.y, e = p.c.indices[pair];
  if (e < 0 || e >= p.c.E || c0 >= p.I) return;
  const int H = p.c.H;
  const uint16_t* g = p.gate_up + (static_cast<int64_t>(e) * 2 * p.I + c0) * H;  // (I is a multiple of 8)
  const uint16_t* const w[4] = {g, g + H, g + static_cast<int64_t>(p.I) * H, g + (static_cast<int64_t>(p.I) + 1) * H};
  float s[1][4];
  dot_rows<1, 4>(p.x + pair / p.c.k * p.ldx, 0, w, H, s);
  if ((threadIdx.x & 63) == 0)
    *reinterpret_cast<uint32_t*>(p.act + static_cast<int64_t>(pair) * p.I + c0) =
        pk_bf16(silu(s[0][0]) * s[0][2], silu(s[0][1]) * s[0][3]);
}

__global__ __launch_bounds__(256) void few_down_kernel(const FewParams p) {
  constexpr int C = 2, CH = 8;  // columns of a wave; loads of 512 values of K on their way
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c0 = (blockIdx.x * 4 + wave) * C, k = p.c.k, I = p.I;
  const int64_t t = blockIdx.y;
  if (c0 >= p.c.H) return;
  const int parts = (I + kLanes8 - 1) / kLanes8, n = k * parts;
  float sum[C] = {};
  for (int s0 = 0; s0 < n; s0 += CH) {
    u32x4 wv[CH][C], av[CH];
    float weight[CH];
#pragma unroll
    for (int s = 0; s < CH; ++s) {
      const int at = min(s0 + s, n - 1), j = at / parts, i = at % parts * kLanes8 + lane * CPL;
      const int e = p.c.indices[t * k + j];
      const bool in = s0 + s < n && e >= 0 && e < p.c.E && i < I;
      weight[s] = in ? p.c.weights[t * k + j] : 0.0f;
      const uint16_t* w = p.down + (static_cast<int64_t>(in ? e : 0) * p.c.H + c0) * I + (in ? i : 0);
      const u32x4 zero = {0u, 0u, 0u, 0u};
      av[s] = zero;
#pragma unroll
      for (int c = 0; c < C; ++c) wv[s][c] = zero;
      if (in) {
        av[s] = *reinterpret_cast<const u32x4*>(p.act + (t * k + j) * I + i);
#pragma unroll
        for (int c = 0; c < C; ++c) wv[s][c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(w + c * I));
      }
    }
#pragma unroll
    for (int s = 0; s < CH; ++s)
#pragma unroll
      for (int c = 0; c < C; ++c) sum[c] += weight[s] * dot8(wv[s][c], av[s], 0.0f);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    sum[c] = wave_sum(sum[c]);
    if (p.c.base) sum[c] += bf16_to_f32(p.c.base[t * p.c.ldb + c0 + c]);
  }
  if (lane == 0) *reinterpret_cast<uint32_t*>(p.c.out + t * p.c.ldo + c0) = pk_bf16(sum[0], sum[1]);
}

// --------------------------------------------------------------------- host

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

// Rows of the experts' tiles.  128 by 256 weight rows use the matrix units and LDS best where the experts have the rows
// for it and the tiles are enough for the CUs, 256 by 256 where they have more of both; us in 64-, 128-, 256-row tiles:
//   2048 x 512, 8 of 256: 512 tokens (16 rows an expert) 290, 315, 345; 1024 (32) 344, 340, 365; 4096 (128) 562, 490, 486
//   1024 x 512, 6 of 64: 1024 (96) 81, 83, 101; 2048 (192) 116, 96, 125; 4096 (384) 179, 159, 142
//   1536 x 1000, 2 of 8: 512 (128; 96 tiles of 128 rows) 42, 52, 75; 4096 (1024) 154, 134, 128
int64_t tile_rows(int64_t P, int64_t I, int64_t E) {
  for (const int64_t rows : {256, 128}) {
    if (P >= (rows == 256 ? 256 : 32) * E && (P / rows + E / 2) * ((I + 127) / 128) >= kCUs) return rows;
  }
  return 64;
}

// Whether the pairs are few: each reads its own weights, without a plan, against those of the experts that are chosen at
// all and a longer way.  Tokens at which the plan becomes the faster one, us without and with it:
//   2048 x 512, 8 of 256: 8 63, 66; 16 125, 107.  4096 x 1536, 4 of 32: 4 96, 104; 8 187, 123 to 138
//   1096 x 328, 3 of 12: 8 15, 20; 16 23.5, 20.5.  1536 x 1000, 2 of 8: 4 16.4, 22.5; 8 26.7, 24.7
// (choices that crowd on some experts, as these did, leave the plan fewer weights to read than the rule expects: at 16
// tokens of the first it still takes the pairs' way)
bool few_pairs(int64_t P, int64_t H, int64_t I, int64_t E) {
  if (P > 1024) return false;
  const double mb = 6e-6 * H * I, chosen = E * (1.0 - std::pow(1.0 - 1.0 / E, static_cast<double>(P)));
  return 5.0 + P * mb / 6.4 < 16.0 + chosen * mb / 5.3;
}

struct ExpertLayout {  // byte offsets in the workspace
  int64_t rows, max_tiles, chunks;
  int64_t tiles, n_tiles, counts, from, to, act, y, nibbles, bytes;
};

ExpertLayout expert_layout(int64_t N, int64_t H, int64_t I, int64_t E, int64_t k) {
  ExpertLayout l = {};
  const int64_t P = N * k;
  l.rows = tile_rows(P, I, E);
  l.max_tiles = P / l.rows + (E < P ? E : P);
  l.chunks = P <= kOneChunk ? 1 : (P + kChunk - 1) / kChunk;
  l.n_tiles = 0;
  l.tiles = 16;
  l.counts = l.tiles + l.max_tiles * sizeof(TileOf);
  l.from = l.counts + round16(l.chunks * E * 4);
  l.to = l.from + round16(P * 4);
  l.act = l.to + round16(P * 4);
  l.y = l.act + P * I * 2;
  l.nibbles = l.y + P * H * 2;
  l.bytes = l.nibbles + P * H / 2;
  return l;
}

// Whether the weights pass by the caches: where an expert has about one tile and the weights would not stay in the 256 MB
// last-level cache until a model's next step in any case (us with and without, 2048 x 512, 8 of 256, 1.6 GB: 64 tokens
// 195, 224; 512 288, 314; 2048 377, 380; but 4096, half of whose experts have a second tile, 523, 489; 1536 x 1000, 2 of 8,
// 74 MB, which the next call finds there, 64 tokens 39, 27).
bool weights_once(int64_t P, int64_t H, int64_t I, int64_t E) {
  return P <= 64 * E && 6e-6 * E * H * I >= 128.0;
}

template <bool PAIR, Store ST>
void launch_experts(const ProductParams& p, const ExpertLayout& l, bool once, hipStream_t st) {
  if (l.rows == 256) launch_product<Large<PAIR>, ST, true>(p, l.max_tiles, st);
  else if (l.rows == 128 && once) launch_product<Wide<PAIR>, ST, true, true>(p, l.max_tiles, st);
  else if (l.rows == 128) launch_product<Wide<PAIR>, ST, true>(p, l.max_tiles, st);
  else if (once) launch_product<Small<PAIR>, ST, true, true>(p, l.max_tiles, st);
  else launch_product<Small<PAIR>, ST, true>(p, l.max_tiles, st);
}

bool expert_sizes_ok(int64_t N, int64_t H, int64_t I, int64_t E, int64_t k) {
  return N >= 0 && H > 0 && I > 0 && E > 0 && E <= kMaxExperts && k > 0 && k <= kMaxChoices && H % 8 == 0 &&
         I % 8 == 0 && H <= INT32_MAX / 4 && I <= INT32_MAX / 4 && N <= (INT32_MAX - 2 * kChunk) / k;
}

// Whether 32-bit byte offsets reach an expert's weights and a tile's inner values.
bool expert_fits(int64_t H, int64_t I) { return weights_fit(2 * I + 256, H) && weights_fit(H, I) && I <= kMostInner; }

}  // namespace

extern "C" size_t gdn_expert_mlp_workspace_bytes(int64_t N, int64_t H, int64_t I, int64_t E, int64_t k) {
  if (!expert_sizes_ok(N, H, I, E, k)) return 0;
  return static_cast<size_t>(expert_layout(N, H, I, E, k).bytes);
}

extern "C" int gdn_expert_mlp_tile_rows(int64_t N, int64_t H, int64_t I, int64_t E, int64_t k) {
  if (!expert_sizes_ok(N, H, I, E, k))
    return gdn_host::fail(GDN_ERR_INVALID, "gdn_expert_mlp_tile_rows: sizes that gdn_expert_mlp does not take");
  if (!expert_fits(H, I)) return gdn_host::fail(GDN_ERR_UNSUPPORTED, "gdn_expert_mlp_tile_rows: weights too large");
  return few_pairs(N * k, H, I, E) ? 0 : static_cast<int>(tile_rows(N * k, I, E));
}

extern "C" int gdn_expert_mlp(const void* x, int64_t ldx, const void* gate_up, const void* down, const int32_t* indices,
                              const float* weights, const void* base, int64_t ldb, void* out, int64_t ldo, int64_t N,
                              int64_t H, int64_t I, int64_t E, int64_t k, void* workspace, size_t workspace_bytes,
                              void* stream) {
  using gdn_host::aligned;
  using gdn_host::fail;
  if (!expert_sizes_ok(N, H, I, E, k))
    return fail(GDN_ERR_INVALID,
                "gdn_expert_mlp: bad sizes N=%lld H=%lld I=%lld E=%lld k=%lld (H and I multiples of 8, E up to %d, k up to %d)",
                (long long)N, (long long)H, (long long)I, (long long)E, (long long)k, kMaxExperts, kMaxChoices);
  if (N == 0) return GDN_OK;
  if (!x || !gate_up || !down || !indices || !weights || !out)
    return fail(GDN_ERR_INVALID, "gdn_expert_mlp: null pointer");
  if (ldx < H || ldo < H || ldx % 8 || ldo % 8 || (base && (ldb < H || ldb % 8)))
    return fail(GDN_ERR_INVALID, "gdn_expert_mlp: row strides must cover the rows and be multiples of 8");
  if (!aligned(x, 16) || !aligned(gate_up, 16) || !aligned(down, 16) || !aligned(out, 16) || !aligned(base, 16) ||
      !aligned(indices, 4) || !aligned(weights, 4))
    return fail(GDN_ERR_INVALID, "gdn_expert_mlp: misaligned pointer");
  if (N > ((int64_t{1} << 30) - H) / ldx + 1)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_expert_mlp: x spans more than 2 GiB (pass fewer tokens a call)");
  if (!expert_fits(H, I))
    return fail(GDN_ERR_UNSUPPORTED, "gdn_expert_mlp: an expert's weights exceed 2 GiB, or I=%lld is over %lld", (long long)I,
                (long long)kMostInner);
  const ExpertLayout l = expert_layout(N, H, I, E, k);
  if (!workspace || workspace_bytes < static_cast<size_t>(l.bytes) || !aligned(workspace, 16))
    return fail(GDN_ERR_INVALID, "gdn_expert_mlp: needs a 16-byte aligned workspace of %lld bytes (got %zu)",
                (long long)l.bytes, workspace_bytes);
  const int64_t widest = l.max_tiles * ((H > I ? H : I) / 64 + 1);
  if (widest > INT32_MAX / 2 || N * (H / 8) / 256 >= INT32_MAX)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_expert_mlp: problem too large");

  const hipStream_t st = static_cast<hipStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  CombineParams c = {};
  c.y = reinterpret_cast<const uint16_t*>(ws + l.y);
  c.nibbles = reinterpret_cast<const uint32_t*>(ws + l.nibbles);
  c.indices = indices;
  c.weights = weights;
  c.base = static_cast<const uint16_t*>(base);
  c.ldb = ldb;
  c.out = static_cast<uint16_t*>(out);
  c.ldo = ldo;
  c.N = N;
  c.H = static_cast<int>(H);
  c.k = static_cast<int>(k);
  c.E = static_cast<int>(E);
  if (few_pairs(N * k, H, I, E)) {
    FewParams f = {};
    f.x = static_cast<const uint16_t*>(x);
    f.ldx = ldx;
    f.gate_up = static_cast<const uint16_t*>(gate_up);
    f.down = static_cast<const uint16_t*>(down);
    f.act = reinterpret_cast<uint16_t*>(ws + l.act);
    f.c = c;
    f.I = static_cast<int>(I);
    hipLaunchKernelGGL(few_up_kernel, dim3(static_cast<unsigned>((I + 7) / 8), static_cast<unsigned>(N * k)), dim3(256), 0,
                       st, f);
    hipLaunchKernelGGL(few_down_kernel, dim3(static_cast<unsigned>((H + 7) / 8), static_cast<unsigned>(N)), dim3(256), 0,
                       st, f);
    return gdn_host::check_launch("gdn_expert_mlp");
  }

  PlanParams plan = {};
  plan.indices = indices;
  plan.P = static_cast<int>(N * k);
  plan.k = static_cast<int>(k);
  plan.E = static_cast<int>(E);
  plan.rows = static_cast<int>(l.rows);
  plan.chunks = static_cast<int>(l.chunks);
  plan.counts = reinterpret_cast<int*>(ws + l.counts);
  plan.tiles = reinterpret_cast<TileOf*>(ws + l.tiles);
  plan.n_tiles = reinterpret_cast<int*>(ws + l.n_tiles);
  plan.from = reinterpret_cast<int*>(ws + l.from);
  plan.to = reinterpret_cast<int*>(ws + l.to);
  const dim3 chunks(static_cast<unsigned>(l.chunks)), threads(kPlanThreads);
  constexpr int kEach = kChunk / kPlanThreads;
  if (l.chunks > 1) {
    hipLaunchKernelGGL(plan_count_kernel, chunks, threads, 0, st, plan);
    hipLaunchKernelGGL(plan_place_kernel<kEach>, chunks, threads, 0, st, plan);
  } else if (plan.P > kChunk) {
    hipLaunchKernelGGL(plan_place_kernel<kOneChunk / kPlanThreads>, chunks, threads, 0, st, plan);
  } else {
    hipLaunchKernelGGL(plan_place_kernel<kEach>, chunks, threads, 0, st, plan);
  }

  const bool once = weights_once(N * k, H, I, E);
  ProductParams p = {};
  p.x = static_cast<const uint16_t*>(x);
  p.ldx = ldx;
  p.w = static_cast<const uint16_t*>(gate_up);
  p.expert_stride = 2 * I * H;
  p.up = static_cast<int>(I);
  p.out = reinterpret_cast<uint16_t*>(ws + l.act);
  p.ldo = I;
  p.N = static_cast<int>(I);
  p.K = static_cast<int>(H);
  p.tiles = plan.tiles;
  p.count = plan.n_tiles;
  p.from = plan.from;
  launch_experts<true, kBare>(p, l, once, st);

  p.x = p.out;
  p.ldx = I;
  p.w = static_cast<const uint16_t*>(down);
  p.expert_stride = H * I;
  p.up = 0;
  p.out = reinterpret_cast<uint16_t*>(ws + l.y);
  p.nibbles = reinterpret_cast<uint32_t*>(ws + l.nibbles);
  p.ldo = H;
  p.N = static_cast<int>(H);
  p.K = static_cast<int>(I);
  p.from = nullptr;
  p.to = plan.to;
  launch_experts<false, kSplit>(p, l, once, st);

  hipLaunchKernelGGL(combine_kernel, dim3(static_cast<unsigned>((N * (H / 8) + 255) / 256)), dim3(256), 0, st, c);
  return gdn_host::check_launch("gdn_expert_mlp");
}
