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

// The tile of the least modelled time: rounds of tiles over the CUs times a tile's fixed part and its steps' (of 64
// values of K, shared by WK groups of waves), which grow with the rows it works on, and below all the operands' bytes at
// the rate the tile reaches.  Fitted to graph-replayed times of 165 sizes (11 products from 512 to 12288 in and 1000 to
// 24576 weight rows, 5 to 4096 rows), each in all four; the choice is the slower one by 0.5% on average, by 16% at most
// (5 to 16 rows of 4096 x 24576: 47 us in the second, 41 in the first).  E.g. 128 rows of 4096 x 4096, us:
// 16.4, 30, 56, 56; 512 of 12288 x 4096: 142, 83, 154, 260; 4096 of 4096 x 24576: 2620, 1285, 700, 619.
struct Tiling {
  int rows, weight_rows, groups, block;  // block: rows that a step's work grows by
  float tile_us, step_us, rows_us;       // a tile's ends, a step, and a step of all rows on top
  float mb_us;                           // MB a us
};
constexpr Tiling kTilings[4] = {
    {64, 32, 4, 16, 3.7f, 0.0f, 0.63f, 3.5f},
    {64, 128, 2, 16, 3.9f, 0.40f, 0.31f, 4.2f},
    {128, 256, 1, 32, 4.0f, 0.40f, 0.40f, 3.1f},
    {256, 256, 1, 32, 4.0f, 0.36f, 1.02f, 3.2f},
};

Tiling tiling(int64_t M, int64_t weight_rows, int64_t K, bool pair) {
  const Tiling* best = nullptr;
  float least = 0.0f;
  for (const Tiling& t : kTilings) {
    const int64_t tiles = ((M + t.rows - 1) / t.rows) * ((weight_rows + t.weight_rows - 1) / t.weight_rows);
    const int64_t whole = (tiles + kCUs - 1) / kCUs;
    const float rounds = whole > 3 ? static_cast<float>(tiles) / kCUs : static_cast<float>(whole);
    int64_t rows = t.block;
    while (rows < t.rows && rows < M) rows *= 2;
    const float steps = static_cast<float>((K + 64 * t.groups - 1) / (64 * t.groups));
    const float mb = 2e-6f * (static_cast<float>(M) * K + static_cast<float>(weight_rows) * K +
                              static_cast<float>(M) * weight_rows / (pair ? 2 : 1));
    float us = rounds * (t.tile_us + steps * (t.step_us + t.rows_us * static_cast<float>(rows) / t.rows));
    us = us > mb / t.mb_us ? us : mb / t.mb_us;
    if (!best || us < least) {
      best = &t;
      least = us;
    }
  }
  return *best;
}

template <bool PAIR>
void launch_tiles(const ProductParams& p, const Tiling& t, int64_t m_tiles, bool bare, hipStream_t st) {
  if (t.rows == 256) {
    if (bare) launch_product<Large<PAIR>, kBare, false>(p, m_tiles, st);
    else launch_product<Large<PAIR>, kFinish, false>(p, m_tiles, st);
  } else if (t.rows == 128) {
    if (bare) launch_product<Wide<PAIR>, kBare, false>(p, m_tiles, st);
    else launch_product<Wide<PAIR>, kFinish, false>(p, m_tiles, st);
  } else if (t.groups == 2) {
    launch_product<Deep<PAIR>, kFinish, false>(p, m_tiles, st);
  } else {
    launch_product<Thin<PAIR>, kFinish, false>(p, m_tiles, st);
  }
}

}  // namespace

extern "C" int gdn_linear_act(const void* x, int64_t ldx, const void* W, const void* bias, int bias_dtype, int act,
                              const void* row_gate, int row_gate_dtype, int64_t ldg, const void* residual, int64_t ldr,
                              void* out, int64_t ldo, int64_t M, int64_t N, int64_t K, void* stream) {
  using gdn_host::aligned;
  using gdn_host::fail;
  if (M < 0 || N <= 0 || K <= 0 || K % 8 || M > INT32_MAX - 256 || N > INT32_MAX / 4)
    return fail(GDN_ERR_INVALID, "gdn_linear_act: bad sizes M=%lld N=%lld K=%lld (K a multiple of 8)", (long long)M,
                (long long)N, (long long)K);
  if (act < GDN_ACT_NONE || act > GDN_ACT_SWIGLU) return fail(GDN_ERR_INVALID, "gdn_linear_act: unknown activation %d", act);
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
  if (!weights_fit(pair ? N + 256 : 256, K) || ldx > (int64_t{1} << 30) / 256 - 64)
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
  if (M <= 4) {
    if (pair) launch_few<true>(p, st);
    else launch_few<false>(p, st);
  } else {
    const bool bare = !bias && !row_gate && !residual && (act == GDN_ACT_NONE || pair);
    const Tiling t = tiling(M, pair ? 2 * N : N, K, pair);
    const int64_t m = (M + t.rows - 1) / t.rows;
    if (pair) launch_tiles<true>(p, t, m, bare, st);
    else launch_tiles<false>(p, t, m, bare, st);
  }
  return gdn_host::check_launch("gdn_linear_act");
}
