// Products of bf16 rows with rows of weights on gfx950 MFMA, with what is done to their sums, shared by the dense ones
// (gdn_linear_act.hip) and the experts' (gdn_experts.hip).
#pragma once

#include <climits>

#include "gdn_common.hpp"

namespace {

using namespace gdn;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kXcds = 8;
constexpr int kCUs = 256;

// What is done with a product's sums before they are rounded (all optional).
struct Epilogue {
  const void* bias;  // [weight rows]
  int bias_dt;
  int act;           // GDN_ACT_*
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
  uint32_t* nibbles;       // kSplit: the sums' next four bits, eight columns a word, rows as out's
  int64_t ldo;
  int M, N, K;             // rows (without a plan), columns of out
  int n_tiles;             // tiles of columns
  // K in slices of `slice` values: slice i's sums go to part + i M pitch, a row's columns (its ups from pitch / 2 on)
  int slices, slice, pitch;
  float* part;
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
    case GDN_ACT_RELU: return x < 0.0f ? 0.0f : x;  // (NaN stays)
    case GDN_ACT_SILU: return silu(x);
    case GDN_ACT_GELU: return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
    case GDN_ACT_GELU_TANH:  // 0.5 x (1 + tanh z) = x sigmoid(2 z)
      return x * sigmoid(1.5957691216057308f * (x + 0.044715f * x * x * x));
    default: return x;
  }
}

// Eight neighbouring bf16 values of which `n` are there, by the widest pieces that their place allows.
__device__ __forceinline__ u32x4 load_bf16x8(const uint16_t* p, int n) {
  if (n >= CPL && reinterpret_cast<uintptr_t>(p) % 16 == 0) return *reinterpret_cast<const u32x4*>(p);
  u32x4 v = {0u, 0u, 0u, 0u};
  if (n >= CPL && reinterpret_cast<uintptr_t>(p) % 4 == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = reinterpret_cast<const uint32_t*>(p)[j];
  } else {
#pragma unroll
    for (int j = 0; j < CPL; ++j)
      if (j < n) v[j / 2] |= static_cast<uint32_t>(p[j]) << (16 * (j % 2));
  }
  return v;
}
__device__ __forceinline__ void store_bf16x8(uint16_t* p, int n, const u32x4& v) {
  if (n >= CPL && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
    *reinterpret_cast<u32x4*>(p) = v;
  } else if (n >= CPL && reinterpret_cast<uintptr_t>(p) % 4 == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) reinterpret_cast<uint32_t*>(p)[j] = v[j];
  } else {
#pragma unroll
    for (int j = 0; j < CPL; ++j)
      if (j < n) p[j] = static_cast<uint16_t>(v[j / 2] >> (16 * (j % 2)));
  }
}

__device__ __forceinline__ void load_bias8(const Epilogue& e, int c, int n, float (&b)[CPL]) {
  if (e.bias_dt == GDN_DTYPE_F32) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) b[j] = j < n ? static_cast<const float*>(e.bias)[c + j] : 0.0f;
  } else {
    const u32x4 v = load_bf16x8(static_cast<const uint16_t*>(e.bias) + c, n);
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const uint16_t h = static_cast<uint16_t>(v[j / 2] >> (16 * (j % 2)));
      b[j] = e.bias_dt == GDN_DTYPE_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
    }
  }
}

// Eight neighbouring columns' sums (of SwiGLU's gates, and its ups) through the epilogue: row `at` of out, columns c on.
template <bool PAIR>
__device__ __forceinline__ void finish8(const ProductParams& p, float (&v)[CPL], float (&up)[CPL], int64_t at, int c) {
  const Epilogue& e = p.epi;
  const int n = p.N - c;  // columns that are there
  // what is read is on its way before the activation
  u32x4 residual = {0u, 0u, 0u, 0u};
  if (e.residual) residual = load_bf16x8(e.residual + at * e.ldr + c, n);
  const float gate = e.gate ? load_any(e.gate, e.gate_dt, at * e.gate_ld) : 0.0f;
  if (e.bias) {
    float b[CPL];
    load_bias8(e, c, n, b);
#pragma unroll
    for (int j = 0; j < CPL; ++j) v[j] += b[j];
    if (PAIR) {
      load_bias8(e, c + p.up, n, b);
#pragma unroll
      for (int j = 0; j < CPL; ++j) up[j] += b[j];
    }
  }
  if constexpr (PAIR) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) v[j] = silu(v[j]) * up[j];
  } else if (e.act == GDN_ACT_GELU) {  // (the others are short: all eight at a time)
#pragma unroll 1
    for (int j = 0; j < CPL; ++j) {  // the values pass by one copy of the code
      const float x = activate(GDN_ACT_GELU, v[0]);
#pragma unroll
      for (int m = 1; m < CPL; ++m) v[m - 1] = v[m];
      v[CPL - 1] = x;
    }
  } else if (e.act == GDN_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) v[j] = activate(GDN_ACT_RELU, v[j]);
  } else if (e.act == GDN_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) v[j] = activate(GDN_ACT_SILU, v[j]);
  } else if (e.act == GDN_ACT_GELU_TANH) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) v[j] = activate(GDN_ACT_GELU_TANH, v[j]);
  }
  if (e.gate) {
    const float g = sigmoid(gate);
#pragma unroll
    for (int j = 0; j < CPL; ++j) v[j] *= g;
  }
  if (e.residual) {
#pragma unroll
    for (int j = 0; j < CPL; ++j)
      v[j] += __uint_as_float(j % 2 ? residual[j / 2] & 0xffff0000u : residual[j / 2] << 16);
  }
  store_bf16x8(p.out + at * p.ldo + c, n,
               u32x4{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]), pk_bf16(v[6], v[7])});
}

// ------------------------------------------------- a sum in 20 bits
//
// An expert's results wait in memory for the sum over a token's experts.  Rounded to bf16 they would be off by as much
// as the output's own rounding is (2^-8 of a column); in fp32 they would be 60% more bytes.  So: the upper 20 bits of the
// fp32 sum, rounded, 16 in a plane of bf16's width and four in a plane of nibbles.  A column is off by at most 2^-12 of itself
// whatever lies beside it.  Half of the last bit is added to all: what carries runs into the exponent, as it should, and
// leaves infinities and NaN as they are (a NaN is a bf16 operand's or the default one, whose lower half is zeros).
__device__ __forceinline__ f32x4 half_added(const f32x4& v) {
  f32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = __uint_as_float(__float_as_uint(v[j]) + 0x800u);
  return r;
}
__device__ __forceinline__ u32x2 upper16(const f32x4& v) {
  return u32x2{__builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x07060302u),
               __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x07060302u)};
}
// The four columns' third bytes, whose upper nibbles count; those of eight columns: column j's is nibble 2 j, 4 + j's 2 j + 1.
__device__ __forceinline__ uint32_t third8(const f32x4& v) {
  return __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x0c0c0501u) |
         __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x05010c0cu);
}
__device__ __forceinline__ uint32_t nibbles8(uint32_t first, uint32_t second) {
  return (first >> 4 & 0x0f0f0f0fu) | (second & 0xf0f0f0f0u);
}
// Four sums back from their upper halves and third bytes.
__device__ __forceinline__ f32x4 joined4(uint32_t lo, uint32_t hi, uint32_t third) {
  return f32x4{__uint_as_float(__builtin_amdgcn_perm(lo, third, 0x0504000cu)),
               __uint_as_float(__builtin_amdgcn_perm(lo, third, 0x0706010cu)),
               __uint_as_float(__builtin_amdgcn_perm(hi, third, 0x0504020cu)),
               __uint_as_float(__builtin_amdgcn_perm(hi, third, 0x0706030cu))};
}

// ------------------------------------------------------------------ product
//
// A tile: up to 16 MB WM rows of x by 16 NB WN rows of W, K in steps of 64.  Both operands' steps go straight into LDS
// (128 bytes a row, all of a cache line).  A step's 16-byte granules lie XOR-swizzled by half their row, so that the 16
// rows that a fragment's read takes at a time lie in all 64 banks.  W is the MFMA's A operand, x its B: a lane's four
// sums are four neighbouring columns of one row.
//
// WM x WN waves share a step and meet once in it: with both halves' fragments of step s in registers, a wave waits for
// its own loads of step s + 1 and for the others; then all have read step s, whose stage the loads of the step that many
// stages on fill while the second half of s is multiplied and s + 1 is.  WK such groups take the steps in turn, each
// with stages of its own, and sum up in LDS at the end.
template <int NB_, int WM_, int WN_, int WK_, int MAXB_, int BY_, int LDS_, bool PAIR_>
struct Shape {
  static constexpr int NB = NB_, WM = WM_, WN = WN_, WK = WK_, MAXB = MAXB_, BY = BY_;
  static constexpr bool PAIR = PAIR_;             // the tile's weight rows are columns' gates and ups
  static constexpr int NG = WM * WN;              // waves of a group
  static constexpr int NT = 64 * NG * WK;         // threads
  static constexpr int WR = 16 * NB * WN;         // weight rows
  static constexpr int COLS = PAIR ? WR / 2 : WR;  // columns of out
  static constexpr int ROWS = 16 * MAXB * WM;      // most rows of x
  static constexpr int LDS = LDS_ * 1024;
};

// Where the buffer loads of steps past K point: no buffer is as long.
constexpr uint32_t kOutside = 0x80000000u;
constexpr uint32_t kWhole = 0x7fffffffu;

// f(A), ..., f(B - 1), each with its number as a constant.
template <int A, int B, class F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (A < B) {
    f(std::integral_constant<int, A>{});
    unrolled<A + 1, B>(f);
  }
}

template <int N>
__device__ __forceinline__ void wait_loads() {  // until at most N loads are on their way
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

enum Store {
  kBare,    // SwiGLU or nothing, to bf16
  kSplit,   // nothing, a sum in 20 bits (N and ldo multiples of 8)
  kFinish,  // all of the epilogue
  kPart,    // a slice of K's sums, as they are
};

// The epilogue of a tile's sums: lane (lr, lq) holds columns 4 lq + 0..3 of its 16-column blocks of row lr of its 16-row
// blocks.  Where nothing but SwiGLU is to be done, straight from the registers.  The rest goes through LDS, as many rows at
// a time as there is room for, eight neighbouring columns a thread, so that its code stands there once and not for each
// of a lane's up to 128 sums (the experts' second product of 4096 tokens, 2048 x 512, 8 of 256, 246 us with all of it in
// the unrolled stores, 176 without; 188 with the nibbles of its sums).
template <class S, int MB, Store ST>
__device__ __forceinline__ void product_store(const ProductParams& p, f32x4 (&acc)[MB][S::NB], int n0, int row0, int rows,
                                              unsigned char* smem) {
  constexpr int NB = S::NB, WM = S::WM, WK = S::WK, NG = S::NG;
  constexpr int OB = S::PAIR ? NB / 2 : NB;  // a wave's blocks of columns of out
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = wave / NG, wg = wave % NG, wm = wg % WM, wn = wg / WM;
  const int lr = lane & 15, lq = lane >> 4;

  if constexpr (ST == kFinish || (ST == kPart && WK > 1)) {
    constexpr int PITCH = S::WR + 4;  // floats a row
    constexpr int FIT = S::LDS / (WK * 16 * WM * PITCH * 4);  // blocks of rows a wave that there is room for
    constexpr int PB = FIT >= MB ? MB : FIT >= 4 ? 4 : FIT >= 2 ? 2 : 1;
    constexpr int PASS = 16 * WM * PB;  // rows at a time
    static_assert(FIT >= 1 && MB % PB == 0, "the sums fit");
    float* sums = reinterpret_cast<float*>(smem);
    for (int i = 0; i < MB; i += PB) {
      if (16 * WM * i >= rows) break;
      __syncthreads();  // the stages, or the pass before, have been read
      unrolled<0, MB>([&](auto at) {
        constexpr int k = at;
        if (i == k / PB * PB) {
#pragma unroll
          for (int b = 0; b < NB; ++b)
            *reinterpret_cast<f32x4*>(sums + (wk * PASS + 16 * (k % PB * WM + wm) + lr) * PITCH + (wn * NB + b) * 16 + 4 * lq) =
                acc[k][b];
        }
      });
      __syncthreads();
      for (int at = threadIdx.x; at < PASS * S::COLS / CPL; at += S::NT) {
        const int r = at / (S::COLS / CPL), oc = at % (S::COLS / CPL) * CPL;
        const int row = 16 * WM * i + r, c = n0 + oc;
        if (row >= rows || c >= p.N) continue;
        const float* from = sums + r * PITCH + (S::PAIR ? oc / (8 * NB) * (16 * NB) + oc % (8 * NB) : oc);
        float v[CPL], up[CPL];
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          v[j] = from[j];
          up[j] = S::PAIR ? from[8 * NB + j] : 0.0f;
#pragma unroll
          for (int g = 1; g < WK; ++g) {
            v[j] += from[g * PASS * PITCH + j];
            if (S::PAIR) up[j] += from[g * PASS * PITCH + 8 * NB + j];
          }
        }
        if constexpr (ST == kPart) {  // (the pitch's halves hold whole fours)
          float* part = p.part + static_cast<int64_t>(row0 + row) * p.pitch + c;
          const bool both = c + 4 < p.N;
          *reinterpret_cast<f32x4*>(part) = f32x4{v[0], v[1], v[2], v[3]};
          if (both) *reinterpret_cast<f32x4*>(part + 4) = f32x4{v[4], v[5], v[6], v[7]};
          if (S::PAIR) {
            *reinterpret_cast<f32x4*>(part + p.pitch / 2) = f32x4{up[0], up[1], up[2], up[3]};
            if (both) *reinterpret_cast<f32x4*>(part + p.pitch / 2 + 4) = f32x4{up[4], up[5], up[6], up[7]};
          }
        } else {
          finish8<S::PAIR>(p, v, up, p.to ? p.to[row0 + row] : row0 + row, c);
        }
      }
    }
  } else if constexpr (ST == kPart) {
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const int r = 16 * (i * WM + wm) + lr;
      if (r >= rows) continue;
      float* out = p.part + static_cast<int64_t>(row0 + r) * p.pitch;
#pragma unroll
      for (int b = 0; b < NB; ++b) {  // (the pitch's halves hold whole fours)
        const int c = n0 + (wn * OB + b % OB) * 16 + 4 * lq;
        if (c < p.N) *reinterpret_cast<f32x4*>(out + c + (b < OB ? 0 : p.pitch / 2)) = acc[i][b];
      }
    }
  } else {
    static_assert(WK == 1, "groups sum up in LDS");
    const int first = n0 + wn * OB * 16;  // the wave's first column
    // all of the wave's columns are there, and 16 bytes of a row are one store
    const bool whole = OB % 2 == 0 && first + OB * 16 <= p.N && (p.ldo & 7) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
    const bool wide = (p.N & 3) == 0 && (p.ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const int r = 16 * (i * WM + wm) + lr, row = min(r, rows - 1);
      const int64_t at = p.to ? p.to[row0 + row] : row0 + row;
      u32x2 y[OB];  // the blocks' four columns
      uint32_t third[ST == kSplit ? OB : 1];
#pragma unroll
      for (int b = 0; b < OB; ++b) {
        f32x4 v = acc[i][b];
        if constexpr (S::PAIR) {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = silu(v[j]) * acc[i][b + OB][j];
        }
        if constexpr (ST == kSplit) {
          v = half_added(v);
          y[b] = upper16(v);
          third[b] = third8(v);
        } else {
          y[b] = u32x2{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3])};
        }
      }
      uint16_t* out = p.out + at * p.ldo + first;
      uint32_t* nibbles = nullptr;
      if constexpr (ST == kSplit) nibbles = p.nibbles + (at * p.ldo + first) / 8;
      if (whole) {
        // two blocks' halves change hands between the 16-lane rows: a lane then has 8 neighbouring columns of one
#pragma unroll
        for (int b = 0; b + 1 < OB; b += 2) {
          const auto lo = __builtin_amdgcn_permlane16_swap(y[b][0], y[b + 1][0], false, false);
          const auto hi = __builtin_amdgcn_permlane16_swap(y[b][1], y[b + 1][1], false, false);
          if (r < rows)
            *reinterpret_cast<u32x4*>(out + (b + (lq & 1)) * 16 + (lq >> 1) * 8) = u32x4{lo[0], hi[0], lo[1], hi[1]};
          if constexpr (ST == kSplit) {
            const auto t = __builtin_amdgcn_permlane16_swap(third[b], third[b + 1], false, false);
            if (r < rows) nibbles[(b + (lq & 1)) * 2 + (lq >> 1)] = nibbles8(t[0], t[1]);
          }
        }
      } else {
#pragma unroll
        for (int b = 0; b < OB; ++b) {
          const int c = first + b * 16 + 4 * lq;
          uint16_t* o = out + b * 16 + 4 * lq;
          if constexpr (ST == kSplit) {  // of the 16-lane rows' pairs the even one has a word's first four columns
            const auto t = __builtin_amdgcn_permlane16_swap(third[b], third[b], false, false);
            if (r < rows && c < p.N && lq % 2 == 0) nibbles[b * 2 + lq / 2] = nibbles8(t[0], t[1]);
          }
          if (r >= rows || c >= p.N) continue;
          if (wide) {
            *reinterpret_cast<u32x2*>(o) = y[b];
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c + j < p.N) o[j] = static_cast<uint16_t>(y[b][j / 2] >> (16 * (j % 2)));
          }
        }
      }
    }
  }
}

// ONCE: W is read once or a few times soon after each other: it does not stay in the caches.
template <class S, int MB, Store ST, bool ONCE>
__device__ __forceinline__ void product_tile(const ProductParams& p, const uint16_t* w, int n0, int row0, int rows,
                                             unsigned char* smem) {
  const int K = ST == kPart ? min(p.slice, p.K) : p.K;
  constexpr int NB = S::NB, WM = S::WM, WK = S::WK, NG = S::NG, WR = S::WR;
  constexpr int STAGE = (WR + 16 * MB * WM) * 128;      // bytes
  constexpr int FIT = S::LDS / (STAGE * WK), STAGES = FIT < 4 ? FIT : 4;
  constexpr int WI = WR / 8 / NG;                       // loads of W a wave and step (8 rows each)
  constexpr int XL = 2 * MB * WM, XI = (XL + NG - 1) / NG;  // of x, all waves' and a wave's (some twice)
  static_assert(STAGES >= 2 && WR % (8 * NG) == 0, "shape");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = wave / NG, wg = wave % NG, wm = wg % WM, wn = wg / WM;
  const int lr = lane & 15, lq = lane >> 4;

  // Load j fills rows 8 j + r8: in place (lane & 7) of a row the granule (lane & 7) ^ (row / 2 % 8)
  const int r8 = lane >> 3;
  const int granule0 = (lane & 7) ^ (r8 >> 1);
  auto granule = [&](int j) { return granule0 ^ ((j & 1) << 2); };
  const uint32_t kbytes = static_cast<uint32_t>(p.K) * 2;
  uint32_t w_off[WI], x_off[XI];
#pragma unroll
  for (int i = 0; i < WI; ++i) {
    const int j = i * NG + wg, tr = 8 * j + r8;
    int col = tr, up = 0;
    if (S::PAIR) {  // a wave's rows: NB / 2 blocks of gates, then the same columns' ups
      const int of = tr % (16 * NB);
      up = of >= 8 * NB ? p.up : 0;
      col = tr / (16 * NB) * (8 * NB) + of % (8 * NB);
    }
    // (columns past the end repeat the last one and are not stored)
    w_off[i] = static_cast<uint32_t>(min(n0 + col, p.N - 1) - n0 + up) * kbytes + granule(j) * 16;
  }
  const uint16_t* x = p.from ? p.x : p.x + row0 * p.ldx;
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int j = (i * NG + wg) % XL;  // (a wave without a share loads another's: each has as many on its way)
    const int r = min(8 * j + r8, rows - 1);  // (rows past the end repeat the last one)
    const int64_t at = (p.from ? static_cast<int64_t>(p.from[row0 + r]) : r) * p.ldx;
    x_off[i] = static_cast<uint32_t>(at) * 2 + granule(j) * 16;
  }
  unsigned char* stages = smem + wk * (STAGES * STAGE);
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(stages));
  // the group's steps: wk, wk + WK, ... (groups that meet have as many each, which past K are of zeros)
  const int nk = ((K + 63) / 64 - (NG > 1 ? 0 : wk) + WK - 1) / WK;

  const uint16_t* wb = w + static_cast<int64_t>(n0) * p.K;
  auto load_part = [&](int s, int st, auto at) {
    constexpr int i = at;
    const int k0 = (s * WK + wk) * 64;
    const uint32_t base = lds0 + st * STAGE;
    if constexpr (i < WI) {
      const int j = i * NG + wg;
      const uint32_t off = k0 + granule(j) * 8 < K ? w_off[i] : kOutside;
      const uint32_t to = __builtin_amdgcn_readfirstlane(base + j * 1024);
      if (ONCE) lds_dma16_once(buf_words(wb + k0, kWhole), off, to);
      else lds_dma16(buf_words(wb + k0, kWhole), off, to);
    } else {
      const int j = ((i - WI) * NG + wg) % XL;
      lds_dma16(buf_words(x + k0, kWhole), k0 + granule(j) * 8 < K ? x_off[i - WI] : kOutside,
                __builtin_amdgcn_readfirstlane(base + WR * 128 + j * 1024));
    }
  };
  auto meet = [&]() {
    if constexpr (NG > 1) asm volatile("s_barrier" : : : "memory");
  };
  // the fragments of half a step: lane (lr, lq) holds 8 values of K of row lr of each 16-row block
  const int frag = lr * 128 + ((lq ^ ((lr >> 1) & 7)) * 16);
  bf16x8 wf[2][NB], xf[2][MB];
  auto read_part = [&](int st, int h, auto at) {
    constexpr int i = at;
    const unsigned char* base = stages + st * STAGE + (frag ^ (h * 64));
    if constexpr (i < NB)
      wf[h][i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(base + (wn * NB + i) * 2048));
    else
      xf[h][i - NB] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(base + WR * 128 + ((i - NB) * WM + wm) * 2048));
  };
  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[i][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // a half's products, with the other half's reads (of stage rs) and a step's loads spread over them
  auto multiply = [&](int h, int rs, bool more, int s, int ls) {
    __builtin_amdgcn_s_setprio(1);
    unrolled<0, MB>([&](auto at) {
      constexpr int i = at;
      unrolled<i * (NB + MB) / MB, (i + 1) * (NB + MB) / MB>([&](auto r) { read_part(rs, h ^ 1, r); });
      if (more) unrolled<i * (WI + XI) / MB, (i + 1) * (WI + XI) / MB>([&](auto l) { load_part(s, ls, l); });
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[i][b] = mfma16(wf[h][b], xf[h][i], acc[i][b]);
      __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_s_setprio(0);
  };

  // (with WK > 1 and little K a group may have no step)
  unrolled<0, STAGES>([&](auto s) {
    if (s < nk) unrolled<0, WI + XI>([&](auto i) { load_part(s, s, i); });
  });
  if (nk >= STAGES) wait_loads<(STAGES - 1) * (WI + XI)>();
  else wait_loads<0>();
  meet();
  unrolled<0, NB + MB>([&](auto i) { read_part(0, 0, i); });
  int st = 0;
  for (int s = 0; s < nk; ++s) {
    multiply(0, st, false, 0, 0);
    if (s + STAGES <= nk) wait_loads<(STAGES - 2) * (WI + XI)>();
    else wait_loads<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    meet();
    const int next = st + 1 == STAGES ? 0 : st + 1;
    multiply(1, next, s + STAGES < nk, s + STAGES, st);  // (past the last step what is read is not used)
    st = next;
  }
  product_store<S, MB, ST>(p, acc, n0, row0, rows, smem);
}

// Runs the tile with a number of 16-row blocks a wave that holds its rows: MB, 2 MB, 3 MB, ... or (DOUBLE) 2 MB, 4 MB, ...
template <class S, Store ST, bool DOUBLE, bool ONCE, int MB>
__device__ __forceinline__ void product_rows(const ProductParams& p, const uint16_t* w, int n0, int row0, int rows,
                                             unsigned char* smem) {
  constexpr int NEXT = DOUBLE ? 2 * MB : MB + S::BY;
  if constexpr (NEXT <= S::MAXB) {
    if (rows > 16 * S::WM * MB) return product_rows<S, ST, DOUBLE, ONCE, NEXT>(p, w, n0, row0, rows, smem);
  }
  product_tile<S, MB, ST, ONCE>(p, w, n0, row0, rows, smem);
}

// PLAN: an expert's tiles of the plan (whose rows vary), or the M rows of x.
template <class S, Store ST, bool PLAN, bool ONCE>
__global__ __launch_bounds__(S::NT) void product_kernel(ProductParams p) {
  __shared__ __align__(1024) unsigned char smem[S::LDS];
  // Block b normally runs on XCD b % 8: each XCD takes neighbouring tiles, which read the same rows and weights, into
  // its L2.  (What a plan holds is only known here: the launch's blocks past it leave.)
  const uint32_t m_tiles = PLAN ? p.count[0] : (p.M + S::ROWS - 1) / S::ROWS;
  const uint32_t total = m_tiles * p.n_tiles * (ST == kPart ? p.slices : 1);
  const uint32_t per = (total + kXcds - 1) / kXcds, local = blockIdx.x / kXcds;
  uint32_t t = blockIdx.x % kXcds * per + local;
  if (local >= per || t >= total) return;
  if constexpr (ST == kPart) {  // all tiles of a slice before the next one's
    const int slice = static_cast<int>(t / (m_tiles * p.n_tiles)), k0 = slice * p.slice;
    t %= m_tiles * p.n_tiles;
    p.x += k0;
    p.w += k0;
    p.part += static_cast<int64_t>(slice) * p.M * p.pitch;
    p.slice = min(p.slice, p.K - k0);
  }
  if constexpr (PLAN) {
    const TileOf of = p.tiles[t / p.n_tiles];
    product_rows<S, ST, false, ONCE, S::BY>(p, p.w + of.expert * p.expert_stride, static_cast<int>(t % p.n_tiles) * S::COLS,
                                      __builtin_amdgcn_readfirstlane(of.row), __builtin_amdgcn_readfirstlane(of.rows), smem);
  } else {
    // eight tiles of rows by all columns at a time
    const uint32_t band = 8 * p.n_tiles, first = t / band * 8, high = min(m_tiles - first, 8u), in = t % band;
    const int row0 = static_cast<int>(first + in % high) * S::ROWS;
    product_rows<S, ST, true, ONCE, 1>(p, p.w, static_cast<int>(in / high) * S::COLS, row0, min(p.M - row0, S::ROWS), smem);
  }
}

template <class S, Store ST, bool PLAN, bool ONCE = false>
void launch_product(ProductParams p, int64_t m_tiles, hipStream_t st) {
  p.n_tiles = (p.N + S::COLS - 1) / S::COLS;
  const int64_t blocks = (m_tiles * p.n_tiles * (ST == kPart ? p.slices : 1) + kXcds - 1) / kXcds * kXcds;
  hipLaunchKernelGGL((product_kernel<S, ST, PLAN, ONCE>), dim3(static_cast<unsigned>(blocks)), dim3(S::NT), 0, st, p);
}

template <bool PAIR> using Thin = Shape<2, 1, 1, 4, 4, 1, 144, PAIR>;    // 64 rows by 32 weight rows
template <bool PAIR> using Deep = Shape<2, 1, 4, 2, 4, 1, 144, PAIR>;    // 64 by 128
template <bool PAIR> using Small = Shape<2, 1, 4, 1, 4, 1, 72, PAIR>;    // 64 by 128
template <bool PAIR> using Wide = Shape<4, 2, 4, 1, 4, 1, 144, PAIR>;    // 128 by 256
template <bool PAIR> using Large = Shape<4, 2, 4, 1, 8, 2, 160, PAIR>;   // 256 by 256

// Rows of an expert's weights are 32-bit byte offsets from the tile's first one.
bool weights_fit(int64_t rows, int64_t K) { return K <= INT32_MAX / 2 && rows < (int64_t{1} << 31) / (2 * K); }

}  // namespace
