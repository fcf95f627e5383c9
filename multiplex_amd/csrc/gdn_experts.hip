// Products of bf16 rows with rows of weights on gfx950 MFMA, and what stands around them in an MLP:
//
//   gdn_linear_act   out = act(x W^T + b) * sigmoid(row_gate) + residual
//   gdn_expert_mlp   out_t = base_t + sum_j w_tj (silu(x_t G_e^T) * (x_t U_e^T)) D_e^T,  e = indices[t][j]
//
// A sparse MLP's tokens choose k of E experts each, so an expert's products have as many rows as tokens chose it, which
// only the device knows.  The pairs (token, choice) are put in the experts' order (plan_place_kernel), every expert's
// cut into tiles of rows, and one launch runs all tiles of all experts: a workgroup finds its expert, rows and columns
// in the plan.  The launch has as many workgroups as the pairs can need at most; those past the plan's end leave.
// SwiGLU happens in the first product's epilogue (a wave forms a column of the gate and the same column of up), its
// result is rounded to bf16 as the second product's operand, the k results of a token are rounded to bf16 and summed in
// fp32 in the order of its choices: a result does not depend on where a pair came to lie in the plan.
#include <climits>

#include "gdn_common.hpp"

namespace {

using namespace gdn;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kXcds = 8;
constexpr int kMaxExperts = 1024;
constexpr int kMaxChoices = 64;

enum Act { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3, kGeluTanh = 4, kSwiglu = 5 };

// What is done with a product's sums before they are rounded (all optional).
struct Epilogue {
  const void* bias;  // [weight rows]
  int bias_dt;
  int act;
  const void* gate;  // [rows], elements gate_ld apart
  int gate_dt;
  int64_t gate_ld;
  const uint16_t* residual;
  int64_t ldr;
};

struct TileOf {  // rows [row, row + rows) of the plan's order, of one expert
  int expert, row, rows, pad;
};

struct ProductParams {
  const uint16_t* x;
  int64_t ldx;
  const uint16_t* w;       // [experts][weight rows][K]
  int64_t expert_stride;   // elements from an expert's weights to the next's
  int up;                  // SwiGLU: weight rows from a column's gate to its up (0: one row a column)
  uint16_t* out;
  int64_t ldo;
  int M, N, K;             // rows (no plan), columns of out
  int n_tiles;             // tiles of columns
  // a plan: the tiles, how many; row r's row of x is from[r] (NULL: r itself), its row of out to[r] (NULL: r)
  const TileOf* tiles;
  const int* count;
  const int* from;
  const int* to;
  Epilogue epi;
};

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
}

__device__ __forceinline__ float activate(int act, float x) {
  switch (act) {
    case kRelu: return x < 0.0f ? 0.0f : x;  // (NaN stays)
    case kSilu: return silu(x);
    case kGelu: return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
    // 0.5 x (1 + tanh z) = x sigmoid(2 z)
    case kGeluTanh: return x * sigmoid(1.5957691216057308f * (x + 0.044715f * x * x * x));
    default: return x;
  }
}

// ------------------------------------------------------------------ product
//
// A tile: up to 16 MB WM rows of x by 16 NB WN rows of W, by WM x WN waves, K in steps of 64.  Both operands' steps go
// straight into LDS (128 bytes a row, all of a cache line), two stages of them.  A step's 16-byte granules lie
// XOR-swizzled by half their row, so that the 16 rows that a fragment's read takes at a time lie in all 64 banks.
// W is the MFMA's A operand, x its B: a lane's four sums are four neighbouring columns of one row.
//
// One barrier a step: with both halves' fragments of step s in registers, a wave waits for its own loads of step s + 1
// and meets the others; then all have read step s, whose stage the loads of s + 2 fill while the second half of s is
// multiplied and s + 1 is.
template <int NB_, int WM_, int WN_, int MAXB_, bool PAIR_>
struct Shape {
  static constexpr int NB = NB_, WM = WM_, WN = WN_, MAXB = MAXB_;
  static constexpr bool PAIR = PAIR_;             // the tile's weight rows are columns' gates and ups
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int WR = 16 * NB * WN;         // weight rows
  static constexpr int COLS = PAIR ? WR / 2 : WR;  // columns of out
  static constexpr int ROWS = 16 * MAXB * WM;      // most rows of x
  static constexpr int STAGE = (WR + ROWS) * 128;  // bytes
};

// Where the buffer loads of steps past K point: no buffer is as long.
constexpr uint32_t kOutside = 0x80000000u;
constexpr uint32_t kWhole = 0x7fffffffu;

template <class S, int MB>
__device__ __forceinline__ void product_tile(const ProductParams& p, const uint16_t* w, int n0, int row0, int rows,
                                             unsigned char* smem) {
  constexpr int NB = S::NB, WM = S::WM, WN = S::WN, NW = S::NW, WR = S::WR;
  constexpr int WI = WR / 8 / NW;                       // loads of W a wave and step (8 rows each)
  constexpr int XL = 2 * MB * WM, XI = (XL + NW - 1) / NW;  // of x, all waves' and a wave's
  static_assert(WR % (8 * NW) == 0 && NW % 2 == 0, "a wave's loads have one parity");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int lr = lane & 15, lq = lane >> 4;

  // Load j fills rows 8 j + r8; lane's granule there.  (8 j + r8) / 2 mod 8 depends on j by its parity, the wave's.
  const int r8 = lane >> 3;
  const int granule = (lane & 7) ^ ((r8 >> 1) | ((wave & 1) << 2));
  const uint32_t kbytes = static_cast<uint32_t>(p.K) * 2;
  uint32_t w_off[WI], x_off[XI];
#pragma unroll
  for (int i = 0; i < WI; ++i) {
    const int tr = 8 * (i * NW + wave) + r8;
    int col = tr, up = 0;
    if (S::PAIR) {  // a wave's rows: NB / 2 blocks of gates, then the same columns' ups
      const int of = tr % (16 * NB);
      up = of >= 8 * NB ? p.up : 0;
      col = tr / (16 * NB) * (8 * NB) + of % (8 * NB);
    }
    // (columns past the end repeat the last one and are not stored)
    w_off[i] = static_cast<uint32_t>(min(n0 + col, p.N - 1) - n0 + up) * kbytes + granule * 16;
  }
  const uint16_t* x = p.from ? p.x : p.x + row0 * p.ldx;
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int r = min(8 * (i * NW + wave) + r8, rows - 1);  // (rows past the end repeat the last one)
    const int64_t at = (p.from ? static_cast<int64_t>(p.from[row0 + r]) : r) * p.ldx;
    x_off[i] = static_cast<uint32_t>(at) * 2 + granule * 16;
  }
  const uint16_t* wb = w + static_cast<int64_t>(n0) * p.K;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem));
  const int nk = (p.K + 63) / 64;

  auto load = [&](int kb, int st) {
    const bool in = kb * 64 + granule * 8 < p.K;
    const u32x4 wr = buf_words(wb + kb * 64, kWhole), xr = buf_words(x + kb * 64, kWhole);
    const uint32_t base = lds0 + st * S::STAGE;
#pragma unroll
    for (int i = 0; i < WI; ++i)
      lds_dma16(wr, in ? w_off[i] : kOutside, __builtin_amdgcn_readfirstlane(base + (i * NW + wave) * 1024));
#pragma unroll
    for (int i = 0; i < XI; ++i)
      if (XL % NW == 0 || i * NW + wave < XL)
        lds_dma16(xr, in ? x_off[i] : kOutside, __builtin_amdgcn_readfirstlane(base + WR * 128 + (i * NW + wave) * 1024));
  };
  // the fragments of half a step: lane (lr, lq) holds 8 values of K of row lr of each 16-row block
  const int frag = lr * 128 + ((lq ^ ((lr >> 1) & 7)) * 16);
  bf16x8 wf[2][NB], xf[2][MB];
  auto read = [&](int st, int h) {
    const unsigned char* base = smem + st * S::STAGE + (frag ^ (h * 64));
#pragma unroll
    for (int b = 0; b < NB; ++b)
      wf[h][b] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(base + (wn * NB + b) * 2048));
#pragma unroll
    for (int b = 0; b < MB; ++b)
      xf[h][b] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(base + WR * 128 + (b * WM + wm) * 2048));
  };
  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[i][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto multiply = [&](int h) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[i][b] = mfma16(wf[h][b], xf[h][i], acc[i][b]);
  };

  load(0, 0);
  if (nk > 1) {
    load(1, 1);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"(WI + XL / NW) : "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" : : : "memory");
  }
  read(0, 0);
  for (int kb = 0; kb < nk; ++kb) {
    const int st = kb & 1;
    read(st, 1);
    multiply(0);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");
    if (kb + 1 < nk) read(st ^ 1, 0);
    if (kb + 2 < nk) load(kb + 2, st);
    multiply(1);
  }

  // lane (lr, lq) holds columns 4 lq + 0..3 of its blocks of row lr
  constexpr int OB = S::PAIR ? NB / 2 : NB;  // blocks of columns of out
  const Epilogue& e = p.epi;
  const bool wide = (p.N & 3) == 0 && (p.ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0;
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int r = 16 * (i * WM + wm) + lr;
    if (r >= rows) continue;
    const int64_t at = p.to ? p.to[row0 + r] : row0 + r;
    const float g = e.gate ? sigmoid(load_any(e.gate, e.gate_dt, at * e.gate_ld)) : 1.0f;
#pragma unroll
    for (int b = 0; b < OB; ++b) {
      const int c = n0 + (wn * OB + b) * 16 + 4 * lq;
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int cj = min(c + j, p.N - 1);
        float v = acc[i][b][j];
        if (e.bias) v += load_any(e.bias, e.bias_dt, cj);
        if constexpr (S::PAIR) {
          float u = acc[i][b + OB][j];
          if (e.bias) u += load_any(e.bias, e.bias_dt, cj + p.up);
          v = silu(v) * u;
        } else {
          v = activate(e.act, v);
        }
        if (e.gate) v *= g;
        if (e.residual) v += bf16_to_f32(e.residual[at * e.ldr + cj]);
        y[j] = v;
      }
      if (c >= p.N) continue;
      uint16_t* o = p.out + at * p.ldo + c;
      if (wide) {
        *reinterpret_cast<u32x2*>(o) = u32x2{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3])};
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < p.N) o[j] = f32_to_bf16(y[j]);
      }
    }
  }
}

// Runs the tile with as few 16-row blocks a wave as hold its rows.
template <class S, int MB = 1>
__device__ __forceinline__ void product_rows(const ProductParams& p, const uint16_t* w, int n0, int row0, int rows,
                                             unsigned char* smem) {
  if constexpr (MB < S::MAXB) {
    if (rows > 16 * S::WM * MB) return product_rows<S, MB + 1>(p, w, n0, row0, rows, smem);
  }
  product_tile<S, MB>(p, w, n0, row0, rows, smem);
}

template <class S>
__global__ __launch_bounds__(S::NT) void product_kernel(const ProductParams p) {
  __shared__ __align__(1024) unsigned char smem[2 * S::STAGE];
  // Block b normally runs on XCD b % 8: each XCD takes neighbouring tiles, which read the same rows, into its L2.
  const int m_tiles = p.tiles ? p.count[0] : (p.M + S::ROWS - 1) / S::ROWS;
  const int64_t total = static_cast<int64_t>(m_tiles) * p.n_tiles;
  const int64_t per = (total + kXcds - 1) / kXcds, local = blockIdx.x / kXcds;
  const int64_t t = blockIdx.x % kXcds * per + local;
  if (local >= per || t >= total) return;
  if (p.tiles) {
    const TileOf tile = p.tiles[t / p.n_tiles];
    product_rows<S>(p, p.w + tile.expert * p.expert_stride, static_cast<int>(t % p.n_tiles) * S::COLS, tile.row,
                    tile.rows, smem);
  } else {
    // eight tiles of rows by all columns at a time
    const int64_t band = 8ll * p.n_tiles;
    const int first = static_cast<int>(t / band) * 8, high = min(m_tiles - first, 8);
    const int of = static_cast<int>(t % band);
    const int row0 = (first + of % high) * S::ROWS;
    product_rows<S>(p, p.w, of / high * S::COLS, row0, min(p.M - row0, S::ROWS), smem);
  }
}

// -------------------------------------------------------------------- plan
//
// The pairs p = t k + j whose expert is one of the E, in the experts' order (from: their tokens, to: the pairs), and
// the experts' tiles of up to `rows` rows.  A chunk of the pairs is one workgroup's; with several chunks a launch
// before counts each chunk's pairs by expert, so that a workgroup knows what lies in front of its own.  Where a pair
// lies among its expert's goes by the atomics' order, which no result depends on.
constexpr int kPlanThreads = 1024;
constexpr int kChunk = 4096;  // pairs

struct PlanParams {
  const int* indices;
  int P, k, E, rows, chunks;
  int* counts;  // [chunks][E]
  TileOf* tiles;
  int* n_tiles;
  int* from;
  int* to;
};

__device__ __forceinline__ void count_pairs(const PlanParams& p, int* hist) {
  for (int e = threadIdx.x; e < p.E; e += kPlanThreads) hist[e] = 0;
  __syncthreads();
  const int first = blockIdx.x * kChunk, last = min(p.P - first, kChunk) + first;
  for (int i = first + threadIdx.x; i < last; i += kPlanThreads) {
    const int e = p.indices[i];
    if (e >= 0 && e < p.E) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
}

__global__ __launch_bounds__(kPlanThreads) void plan_count_kernel(const PlanParams p) {
  __shared__ int hist[kMaxExperts];
  count_pairs(p, hist);
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

__global__ __launch_bounds__(kPlanThreads) void plan_place_kernel(const PlanParams p) {
  __shared__ int next[kMaxExperts];
  __shared__ int waves[kPlanThreads / 64];
  static_assert(kMaxExperts <= kPlanThreads, "a thread an expert");
  const int e = threadIdx.x;
  int mine = 0, total = 0;  // pairs of expert e in the chunks before, and in all
  if (p.chunks == 1) {
    count_pairs(p, next);
    if (e < p.E) total = next[e];
  } else if (e < p.E) {
    for (int c = 0; c < p.chunks; ++c) {
      const int n = p.counts[c * p.E + e];
      total += n;
      if (c < static_cast<int>(blockIdx.x)) mine += n;
    }
  }
  int all;
  const int first = block_before(total, waves, &all);
  const int tiles = (total + p.rows - 1) / p.rows;
  const int tile0 = block_before(tiles, waves, &all);
  if (e < p.E) next[e] = first + mine;
  if (blockIdx.x == 0) {
    for (int i = 0; i < tiles; ++i)
      p.tiles[tile0 + i] = TileOf{e, first + i * p.rows, min(p.rows, total - i * p.rows), 0};
    if (e == 0) p.n_tiles[0] = all;
  }
  __syncthreads();
  const int begin = blockIdx.x * kChunk, end = min(p.P - begin, kChunk) + begin;
  for (int i = begin + threadIdx.x; i < end; i += kPlanThreads) {
    const int x = p.indices[i];
    if (x >= 0 && x < p.E) {
      const int at = atomicAdd(&next[x], 1);
      p.from[at] = i / p.k;
      p.to[at] = i;
    }
  }
}

// ------------------------------------------------------------------- combine

struct CombineParams {
  const uint16_t* y;  // [N k][H]
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
  for (int j = 0; j < p.k; ++j) {
    const int e = p.indices[t * p.k + j];
    if (e < 0 || e >= p.E) continue;
    const float w = p.weights[t * p.k + j];
    float y[CPL];
    unpack8<GDN_DTYPE_BF16>(load_raw8<GDN_DTYPE_BF16>(p.y, (t * p.k + j) * p.H + c), y);
#pragma unroll
    for (int m = 0; m < CPL; ++m) sum[m] += w * y[m];
  }
  store8<GDN_DTYPE_BF16>(p.out, t * p.ldo + c, sum);
}

// --------------------------------------------------------------------- host

using Small = Shape<2, 1, 4, 4, false>;
using SmallPair = Shape<2, 1, 4, 4, true>;

template <class S>
void launch_product(ProductParams p, int64_t m_tiles, hipStream_t st) {
  p.n_tiles = (p.N + S::COLS - 1) / S::COLS;
  const int64_t blocks = (m_tiles * p.n_tiles + kXcds - 1) / kXcds * kXcds;
  hipLaunchKernelGGL(product_kernel<S>, dim3(static_cast<unsigned>(blocks)), dim3(S::NT), 0, st, p);
}

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

struct ExpertLayout {  // byte offsets in the workspace
  int64_t rows, max_tiles, chunks;
  int64_t tiles, n_tiles, counts, from, to, act, y, bytes;
};

ExpertLayout expert_layout(int64_t N, int64_t H, int64_t I, int64_t E, int64_t k) {
  ExpertLayout l = {};
  const int64_t P = N * k;
  l.rows = Small::ROWS;
  l.max_tiles = P / l.rows + (E < P ? E : P);
  l.chunks = (P + kChunk - 1) / kChunk;
  l.n_tiles = 0;
  l.tiles = 16;
  l.counts = l.tiles + l.max_tiles * sizeof(TileOf);
  l.from = l.counts + round16(l.chunks * E * 4);
  l.to = l.from + round16(P * 4);
  l.act = l.to + round16(P * 4);
  l.y = l.act + P * I * 2;
  l.bytes = l.y + P * H * 2;
  return l;
}

bool expert_sizes_ok(int64_t N, int64_t H, int64_t I, int64_t E, int64_t k) {
  return N >= 0 && H > 0 && I > 0 && E > 0 && E <= kMaxExperts && k > 0 && k <= kMaxChoices && H % 8 == 0 &&
         I % 8 == 0 && H <= INT32_MAX / 4 && I <= INT32_MAX / 4 && N <= INT32_MAX / k;
}

// Rows of an expert's weights are 32-bit byte offsets from the tile's first one.
bool weights_fit(int64_t rows, int64_t K) { return K <= INT32_MAX / 2 && rows < (int64_t{1} << 31) / (2 * K); }

}  // namespace

extern "C" size_t gdn_expert_mlp_workspace_bytes(int64_t N, int64_t H, int64_t I, int64_t E, int64_t k) {
  if (!expert_sizes_ok(N, H, I, E, k)) return 0;
  return static_cast<size_t>(expert_layout(N, H, I, E, k).bytes);
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
  if (!weights_fit(2 * I + 256, H) || !weights_fit(H, I))
    return fail(GDN_ERR_UNSUPPORTED, "gdn_expert_mlp: an expert's weights exceed 2 GiB");
  const ExpertLayout l = expert_layout(N, H, I, E, k);
  if (!workspace || workspace_bytes < static_cast<size_t>(l.bytes) || !aligned(workspace, 16))
    return fail(GDN_ERR_INVALID, "gdn_expert_mlp: needs a 16-byte aligned workspace of %lld bytes (got %zu)",
                (long long)l.bytes, workspace_bytes);
  const int64_t widest = l.max_tiles * ((H > I ? H : I) / 64 + 1);
  if (widest > INT32_MAX / 2 || N * (H / 8) / 256 >= INT32_MAX)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_expert_mlp: problem too large");

  const hipStream_t st = static_cast<hipStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
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
  const dim3 chunks(static_cast<unsigned>(l.chunks));
  if (l.chunks > 1) hipLaunchKernelGGL(plan_count_kernel, chunks, dim3(kPlanThreads), 0, st, plan);
  hipLaunchKernelGGL(plan_place_kernel, chunks, dim3(kPlanThreads), 0, st, plan);

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
  launch_product<SmallPair>(p, l.max_tiles, st);

  p.x = p.out;
  p.ldx = I;
  p.w = static_cast<const uint16_t*>(down);
  p.expert_stride = H * I;
  p.up = 0;
  p.out = reinterpret_cast<uint16_t*>(ws + l.y);
  p.ldo = H;
  p.N = static_cast<int>(H);
  p.K = static_cast<int>(I);
  p.from = nullptr;
  p.to = plan.to;
  launch_product<Small>(p, l.max_tiles, st);

  CombineParams c = {};
  c.y = p.out;
  c.indices = indices;
  c.weights = weights;
  c.base = static_cast<const uint16_t*>(base);
  c.ldb = ldb;
  c.out = static_cast<uint16_t*>(out);
  c.ldo = ldo;
  c.N = N;
  c.H = static_cast<int>(H);
  c.k = plan.k;
  c.E = plan.E;
  hipLaunchKernelGGL(combine_kernel, dim3(static_cast<unsigned>((N * (H / 8) + 255) / 256)), dim3(256), 0, st, c);
  return gdn_host::check_launch("gdn_expert_mlp");
}

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
  if ((M / Small::ROWS + 1) * (N / 64 + 1) > INT32_MAX / 2)
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
  const int64_t m_tiles = (M + Small::ROWS - 1) / Small::ROWS;
  if (pair) launch_product<SmallPair>(p, m_tiles, st);
  else launch_product<Small>(p, m_tiles, st);
  return gdn_host::check_launch("gdn_linear_act");
}
