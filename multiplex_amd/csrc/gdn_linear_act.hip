// out = act(x W^T + b) * sigmoid(row_gate) + residual (gdn_linear_act).
#include "gdn_dot.hpp"

namespace {

// R rows of x (all that there are); a wave's W rows of weights are W columns, or the gates and ups of W / 2.
template <int R, int W, bool PAIR>
__global__ __launch_bounds__(256) void few_rows_kernel(const ProductParams p) {
  constexpr int C = PAIR ? W / 2 : W;
  const int lane = threadIdx.x & 63;
  const int c0 = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * C;
  if (c0 >= p.N) return;
  const uint16_t* w[W];
#pragma unroll
  for (int i = 0; i < W; ++i) w[i] = p.w + (static_cast<int64_t>(min(c0 + i % C, p.N - 1)) + (i < C ? 0 : p.up)) * p.K;
  float sums[R][W];
  dot_rows<R, W>(p.x, p.ldx, w, p.K, sums);
  // lane r C + c finishes row r's column c
  float v = 0.0f, u = 0.0f;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (lane != r * C + c) continue;
      v = sums[r][c];
      if (PAIR) u = sums[r][c + C];
    }
  const int row = lane / C, c = c0 + lane % C;
  if (row >= R || c >= p.N) return;
  const Epilogue& e = p.epi;
  if (e.bias) v += load_any(e.bias, e.bias_dt, c);
  if (PAIR) {
    if (e.bias) u += load_any(e.bias, e.bias_dt, c + p.up);
    v = silu(v) * u;
  } else {
    v = activate(e.act, v);
  }
  if (e.gate) v *= sigmoid(load_any(e.gate, e.gate_dt, row * e.gate_ld));
  if (e.residual) v += bf16_to_f32(e.residual[row * e.ldr + c]);
  p.out[row * p.ldo + c] = f32_to_bf16(v);
}

template <int R, bool PAIR>
void launch_few(const ProductParams& p, hipStream_t st) {
  // two weight rows a wave where four would leave CUs without one
  const bool two = p.N * (PAIR ? 2 : 1) <= 2 * 4 * 4 * 256;
  const int cols = (two ? 2 : 4) / (PAIR ? 2 : 1) * 4;
  const dim3 grid(static_cast<unsigned>((p.N + cols - 1) / cols));
  if (two) hipLaunchKernelGGL((few_rows_kernel<R, 2, PAIR>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((few_rows_kernel<R, 4, PAIR>), grid, dim3(256), 0, st, p);
}

template <bool PAIR>
void launch_few(const ProductParams& p, hipStream_t st) {
  switch (p.M) {
    case 1: return launch_few<1, PAIR>(p, st);
    case 2: return launch_few<2, PAIR>(p, st);
    case 3: return launch_few<3, PAIR>(p, st);
    default: return launch_few<4, PAIR>(p, st);
  }
}

}  // namespace

namespace {

// The sum of the slices' sums and the epilogue, eight columns of a row a thread.  Bound by reading the sums.
template <bool PAIR>
__global__ __launch_bounds__(256) void finish_kernel(const ProductParams p) {
  const int per = (p.N + CPL - 1) / CPL;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, row = i / per;
  if (row >= p.M) return;
  const int c = static_cast<int>(i % per) * CPL;
  float v[CPL] = {}, up[CPL] = {};
  auto add = [](float (&sum)[CPL], const float* at, bool both) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h && !both) break;
      const f32x4 x = *reinterpret_cast<const f32x4*>(at + 4 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[4 * h + j] += x[j];
    }
  };
  const float* at = p.part + row * p.pitch + c;
  const bool both = c + 4 < p.N;  // (the pitch's halves hold whole fours)
  for (int s = 0; s < p.slices; ++s, at += static_cast<int64_t>(p.M) * p.pitch) {
    add(v, at, both);
    if (PAIR) add(up, at + p.pitch / 2, both);
  }
  finish8<PAIR>(p, v, up, row, c);
}

// The tile and slices of K of the least modelled time: rounds of tiles over the CUs times a tile's fixed part and its
// steps' (of 64 values of K, shared by the groups of waves), which grow with the rows it works on, the slices' sums
// written and read, and below all the operands' bytes at the rate that the tile reaches.  Where K is no multiple of 64,
// rows start inside cache lines and a step's loads take two lines a row.  Fitted to graph-replayed times of 140 sizes (16
// products from 512 to 12288 in and 700 to 24576 weight rows, seven of them with such K; 8 to 4096 rows) in up to 12
// ways each; the choice is 2.8% slower than the best of them on average, at most 59% (8 x 3320 x 9244: 31 us in the second
// tile, 20 in the first).  E.g. 128 rows of 4096 x 4096, us in the four tiles: 16.4, 30, 56, 56; 512 of 12288 x 4096: 142,
// 83, 154, 260; 4096 of 4096 x 24576: 2620, 1285, 700, 619.  Slices of K pay where a few tiles have many steps: 512 of
// 12288 x 4096 in 4 slices 62, 128 of them in 8 41, 1024 of 4096 x 4096 in 2 46 (53 whole).
struct Tiling {
  int rows, weight_rows, groups, block;  // block: rows that a step's work grows by
  float tile_us, step_us, rows_us;       // a tile's ends, a step, and a step of all rows on top
  float mb_us;                           // MB a us
  float across_step, across_mb;          // what step_us and mb_us are times where rows start inside lines
  int slices;
};
constexpr Tiling kTilings[4] = {
    {64, 32, 4, 16, 1.6f, 0.28f, 0.40f, 3.5f, 1.48f, 0.71f, 1},
    {64, 128, 2, 16, 2.2f, 0.52f, 0.24f, 4.1f, 1.50f, 0.72f, 1},
    {128, 256, 1, 32, 2.9f, 0.46f, 0.38f, 4.0f, 1.67f, 0.73f, 1},
    {256, 256, 1, 32, 3.2f, 0.40f, 1.04f, 4.0f, 1.82f, 0.74f, 1},
};
constexpr float kFinishUs = 5.5f, kPartMbUs = 6.1f;  // the slices' launch, and MB of their sums a us

Tiling tiling(int64_t M, int64_t N, int64_t K, bool pair) {
  const int64_t weight_rows = pair ? 2 * N : N;
  const float mb = 2e-6f * (static_cast<float>(M) * K + static_cast<float>(weight_rows) * K + static_cast<float>(M) * N);
  const bool across = K % 64 != 0;
  Tiling best = kTilings[0];
  float least = 0.0f;
  bool any = false;
  for (const Tiling& t : kTilings) {
    const float step_us = t.step_us * (across ? t.across_step : 1.0f), mb_us = t.mb_us * (across ? t.across_mb : 1.0f);
    for (int slices = 1; slices <= 8; slices *= 2) {
      const int64_t steps = ((K + 64 * t.groups - 1) / (64 * t.groups) + slices - 1) / slices;
      // (as few steps, and as many slices of the tiles whose groups share K, as were measured)
      if (slices > 1 && (steps * t.groups < 16 || slices > (t.groups > 1 ? 4 : 8) ||
                         M * weight_rows > (int64_t{1} << 28)))
        break;
      const int64_t tiles = ((M + t.rows - 1) / t.rows) * ((weight_rows + t.weight_rows - 1) / t.weight_rows) * slices;
      const int64_t whole = (tiles + kCUs - 1) / kCUs;
      const float rounds = whole > 3 ? static_cast<float>(tiles) / kCUs : static_cast<float>(whole);
      int64_t rows = t.block;
      while (rows < t.rows && rows < M) rows *= 2;
      float us = rounds * (t.tile_us + steps * (step_us + t.rows_us * static_cast<float>(rows) / t.rows));
      us = us > mb / mb_us ? us : mb / mb_us;
      if (slices > 1) us += kFinishUs + 8e-6f * slices * M * weight_rows / kPartMbUs;
      if (any && us >= least) continue;
      any = true;
      least = us;
      best = t;
      best.slices = slices;
    }
  }
  return best;
}

constexpr int kFewRows = 4;

// Values of K a slice (whole steps), and how many slices hold any.
int64_t slice_values(const Tiling& t, int64_t K) { return ((K + 63) / 64 + t.slices - 1) / t.slices * 64; }
int slices_of(const Tiling& t, int64_t K) {
  return static_cast<int>((K + slice_values(t, K) - 1) / slice_values(t, K));
}

int64_t part_pitch(int64_t N, bool pair) { return (N + 3) / 4 * 4 * (pair ? 2 : 1); }

int64_t part_bytes(int64_t M, int64_t N, int64_t K, bool pair) {
  if (M <= kFewRows) return 0;
  const Tiling t = tiling(M, N, K, pair);
  return t.slices > 1 ? 4 * t.slices * M * part_pitch(N, pair) : 0;
}

template <class S, bool PAIR>
void launch_slices(const ProductParams& p, int64_t m_tiles, hipStream_t st) {
  launch_product<S, kPart, false>(p, m_tiles, st);
  const int64_t threads = static_cast<int64_t>(p.M) * ((p.N + CPL - 1) / CPL);
  hipLaunchKernelGGL((finish_kernel<PAIR>), dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, st, p);
}

template <bool PAIR>
void launch_tiles(const ProductParams& p, const Tiling& t, bool bare, hipStream_t st) {
  const int64_t m_tiles = (p.M + t.rows - 1) / t.rows;
  if (t.rows == 256) {
    if (t.slices > 1) launch_slices<Large<PAIR>, PAIR>(p, m_tiles, st);
    else if (bare) launch_product<Large<PAIR>, kBare, false>(p, m_tiles, st);
    else launch_product<Large<PAIR>, kFinish, false>(p, m_tiles, st);
  } else if (t.rows == 128) {
    if (t.slices > 1) launch_slices<Wide<PAIR>, PAIR>(p, m_tiles, st);
    else if (bare) launch_product<Wide<PAIR>, kBare, false>(p, m_tiles, st);
    else launch_product<Wide<PAIR>, kFinish, false>(p, m_tiles, st);
  } else if (t.groups == 2) {
    if (t.slices > 1) launch_slices<Deep<PAIR>, PAIR>(p, m_tiles, st);
    else launch_product<Deep<PAIR>, kFinish, false>(p, m_tiles, st);
  } else {
    if (t.slices > 1) launch_slices<Thin<PAIR>, PAIR>(p, m_tiles, st);
    else launch_product<Thin<PAIR>, kFinish, false>(p, m_tiles, st);
  }
}

bool linear_sizes_ok(int64_t M, int64_t N, int64_t K, int act) {
  return M >= 0 && N > 0 && K > 0 && K % 8 == 0 && M <= INT32_MAX - 256 && N <= INT32_MAX / 4 && K <= INT32_MAX / 2 &&
         act >= GDN_ACT_NONE && act <= GDN_ACT_SWIGLU;
}

// Whether 32-bit byte offsets reach a tile's weights.
bool linear_fits(int64_t N, int64_t K, int act) { return weights_fit(act == GDN_ACT_SWIGLU ? N + 256 : 256, K); }

}  // namespace

extern "C" size_t gdn_linear_act_workspace_bytes(int64_t M, int64_t N, int64_t K, int act) {
  return linear_sizes_ok(M, N, K, act) ? static_cast<size_t>(part_bytes(M, N, K, act == GDN_ACT_SWIGLU)) : 0;
}

extern "C" int gdn_linear_act_tile(int64_t M, int64_t N, int64_t K, int act, int32_t* tile) {
  if (!linear_sizes_ok(M, N, K, act) || !tile)
    return gdn_host::fail(GDN_ERR_INVALID, "gdn_linear_act_tile: sizes that gdn_linear_act does not take, or no place");
  if (!linear_fits(N, K, act))
    return gdn_host::fail(GDN_ERR_UNSUPPORTED, "gdn_linear_act_tile: rows too long");
  tile[0] = tile[1] = tile[2] = 0;
  if (M <= kFewRows) return GDN_OK;
  const Tiling t = tiling(M, N, K, act == GDN_ACT_SWIGLU);
  tile[0] = t.rows;
  tile[1] = t.weight_rows;
  tile[2] = slices_of(t, K);
  return GDN_OK;
}

extern "C" int gdn_linear_act(const void* x, int64_t ldx, const void* W, const void* bias, int bias_dtype, int act,
                              const void* row_gate, int row_gate_dtype, int64_t ldg, const void* residual, int64_t ldr,
                              void* out, int64_t ldo, int64_t M, int64_t N, int64_t K, void* workspace,
                              size_t workspace_bytes, void* stream) {
  using gdn_host::aligned;
  using gdn_host::fail;
  if (!linear_sizes_ok(M, N, K, act))
    return fail(GDN_ERR_INVALID, "gdn_linear_act: bad sizes M=%lld N=%lld K=%lld (K a multiple of 8) or activation %d",
                (long long)M, (long long)N, (long long)K, act);
  if (M == 0) return GDN_OK;
  if (!x || !W || !out) return fail(GDN_ERR_INVALID, "gdn_linear_act: null pointer");
  if ((bias && !gdn_host::dtype_ok(bias_dtype)) || (row_gate && !gdn_host::dtype_ok(row_gate_dtype)))
    return fail(GDN_ERR_INVALID, "gdn_linear_act: unknown dtype");
  if (ldx < K || ldx % 8 || ldo < N || (residual && ldr < N) || (row_gate && ldg < 0))
    return fail(GDN_ERR_INVALID, "gdn_linear_act: row strides must cover the rows (x's a multiple of 8)");
  const auto size = [](int dt) { return dt == GDN_DTYPE_F32 ? 4 : 2; };
  if (!aligned(x, 16) || !aligned(W, 16) || !aligned(out, 2) || !aligned(residual, 2) ||
      !aligned(bias, size(bias_dtype)) || !aligned(row_gate, size(row_gate_dtype)))
    return fail(GDN_ERR_INVALID, "gdn_linear_act: misaligned pointer");
  const bool pair = act == GDN_ACT_SWIGLU;
  if (!linear_fits(N, K, act) || ldx > (int64_t{1} << 30) / 256 - 64)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_linear_act: rows too long");
  if ((M / 64 + 1) * (N / 16 + 1) > INT32_MAX / 2)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_linear_act: problem too large");
  ProductParams p = {};
  p.x = static_cast<const uint16_t*>(x);
  p.ldx = ldx;
  p.w = static_cast<const uint16_t*>(W);
  p.up = pair ? static_cast<int>(N) : 0;
  p.out = static_cast<uint16_t*>(out);
  p.ldo = ldo;
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.epi.bias = bias;
  p.epi.bias_dt = bias_dtype;
  p.epi.act = act;
  p.epi.gate = row_gate;
  p.epi.gate_dt = row_gate_dtype;
  p.epi.gate_ld = ldg;
  p.epi.residual = static_cast<const uint16_t*>(residual);
  p.epi.ldr = ldr;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool bare = !bias && !row_gate && !residual && (act == GDN_ACT_NONE || pair);
  // up to four rows: 12288 x 4096 at one 18.3 us (as tiles 25.8), at four 24.4 (27.2); 2048 x 1024 3.8 (4.8), 4.5 (4.8)
  if (M <= kFewRows) {
    if (pair) launch_few<true>(p, st);
    else launch_few<false>(p, st);
    return gdn_host::check_launch("gdn_linear_act");
  }
  const Tiling t = tiling(M, N, K, pair);
  if (t.slices > 1) {
    const int64_t need = part_bytes(M, N, K, pair);
    if (!workspace || workspace_bytes < static_cast<size_t>(need) || !aligned(workspace, 16))
      return fail(GDN_ERR_INVALID, "gdn_linear_act: needs a 16-byte aligned workspace of %lld bytes (got %zu)",
                  (long long)need, workspace_bytes);
    p.slices = slices_of(t, K);
    p.slice = static_cast<int>(slice_values(t, K));
    p.pitch = static_cast<int>(part_pitch(N, pair));
    p.part = static_cast<float*>(workspace);
  }
  if (pair) launch_tiles<true>(p, t, bare, st);
  else launch_tiles<false>(p, t, bare, st);
  return gdn_host::check_launch("gdn_linear_act");
}
