// The paged key/value cache of the full-attention layers on gfx950.
//
//   tables_kernel        block tables, slots and the free list from the rows'
//                        lengths and their new tokens.
//   attn_rope_kernel     RMSNorm of q and k over the head dim, rotary positions
//                        from a table of frequencies (half or interleaved
//                        pairs), q out, k and v into their slots.
//   attention            the kernels of gdn_attention.hpp over the tables: the
//                        keys that all rows share once for the whole batch, each
//                        row's own, and the partial results merged.
#include <algorithm>

#include "gdn_attention.hpp"

namespace {

// ------------------------------------------------------------ tables

struct TableParams {
  const int32_t* lengths;  // [B]
  const int32_t* n_new;    // [B] or null: T
  int32_t* table;          // [B, table_ld]
  const int32_t* held;     // [B] blocks a row's table lists
  int32_t* free;           // [n_blocks] stack of free blocks
  const int32_t* n_free;   // [1]
  int32_t* held_out;
  int32_t* n_free_out;
  int32_t* slots;  // [B, T]
  int B, T, table_ld, lg, shared, n_blocks;
};

constexpr int kTableRows = 4096, kTableThreads = 1024;

// The last of n ascending entries that is not above x (entry 0 is not).
__device__ __forceinline__ int last_not_above(const int32_t* at, int n, int x) {
  int lo = 0;
  for (int hi = n; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Inclusive sum over the lanes up to this one, by DPP moves: in rows of 16, then row 0's and
// row 2's last lane to the row above, then lane 31's to the upper half.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // row_shr 1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, true);  // row_bcast 15, to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, true);  // row_bcast 31, to rows 2 and 3
  return x;
}

// Row b needs max(ceil((len + new) / block), shared) blocks.  Rows with more
// give the last ones back, onto the free stack's top in row order, then rows
// with fewer take from the top in row order, as far as the stack reaches: a row
// that does not get all it asks for gets none, and no row after it any.
// Every workgroup forms the running sums of all rows by itself (PER rows a
// thread) and then takes its share of the cells; a cell that one writes, none
// reads: blocks given back in this call are taken from their giver's table, not
// from the stack.  State that would be written over what other workgroups read
// (held_out = held) is written by a launch of one workgroup (kState) behind the
// others (kCells).
// Bound by latency: the launch, the rows' loads, two barriers, and the table's or
// the stack's loads, of which a thread's first is asked for before the sums
// (256 rows of one token 6.2 us graph-replayed, 1000 of up to nine 8.1; the first
// form, which formed a row anew wherever it was needed and summed in 64 bits, 9.5
// and 10.7).
constexpr int kCells = 1, kState = 2;
template <int PER>
__global__ __launch_bounds__(kTableThreads) void tables_kernel(const TableParams p, int what) {
  constexpr int NW = kTableThreads / 64;
  // of each row: what goes before it, its blocks now and then, its length and (where served) new tokens
  __shared__ int32_t back_at[PER * kTableThreads + 1], take_at[PER * kTableThreads + 1];
  __shared__ int32_t row_have[PER * kTableThreads], row_want[PER * kTableThreads];
  __shared__ int32_t row_len[PER * kTableThreads], row_new[PER * kTableThreads];
  __shared__ int32_t wave_back[NW], wave_take[NW], wave_granted[NW];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n_slots = static_cast<int64_t>(p.B) * p.T;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kTableThreads + tid, step = gridDim.x * kTableThreads;

  int len[PER], fresh[PER], have[PER], want[PER];
  bool fits[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = min(PER * tid + k, p.B - 1);
    len[k] = p.lengths[b];
    fresh[k] = p.n_new != nullptr ? p.n_new[b] : p.T;
    have[k] = p.held[b];
  }
  const int n_free = min(max(p.n_free[0], 0), p.n_blocks);
  // the block that the table lists now at the thread's first token, if it is one of the row's
  int32_t first_block = 0;
  if ((what & kCells) && first < n_slots && p.table_ld > 0) {
    const int b = static_cast<int>(first / p.T), t = static_cast<int>(first - static_cast<int64_t>(b) * p.T);
    const int64_t c = (static_cast<int64_t>(max(p.lengths[b], 0)) + t) >> p.lg;
    first_block = p.table[static_cast<int64_t>(b) * p.table_ld + (c < p.table_ld ? c : p.table_ld - 1)];
  }
  int back = 0, take = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const bool row = PER * tid + k < p.B;
    len[k] = max(len[k], 0);
    fresh[k] = min(max(fresh[k], 0), p.T);
    have[k] = row ? min(max(have[k], 0), p.table_ld) : 0;
    const int64_t need =
        max<int64_t>((static_cast<int64_t>(len[k]) + fresh[k] + (int64_t(1) << p.lg) - 1) >> p.lg, p.shared);
    fits[k] = need <= p.table_ld;
    want[k] = row && fits[k] ? static_cast<int>(need) : have[k];
    back += max(have[k] - want[k], 0);
    take += max(want[k] - have[k], 0);
  }
  const int back_incl = wave_scan(back), take_incl = wave_scan(take);
  if (lane == 63) {
    wave_back[wave] = back_incl;
    wave_take[wave] = take_incl;
  }
  __syncthreads();
  int back_sum = back_incl - back, take_sum = take_incl - take, all_back = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const int x = wave_back[w], y = wave_take[w];
    if (w < wave) {
      back_sum += x;
      take_sum += y;
    }
    all_back += x;
  }
  const int top = static_cast<int>(min<int64_t>(static_cast<int64_t>(n_free) + all_back, INT32_MAX));
  int granted = 0;  // blocks taken by the rows up to this thread's last that takes any
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = PER * tid + k, grow = max(want[k] - have[k], 0);
    const bool served = fits[k] && (grow == 0 || take_sum + grow <= top);
    if (!served) want[k] = have[k];
    if (b < p.B) {
      back_at[b] = back_sum;
      take_at[b] = take_sum;
      row_have[b] = have[k];
      row_want[b] = want[k];
      row_len[b] = len[k];
      row_new[b] = served ? fresh[k] : 0;
    }
    back_sum += max(have[k] - want[k], 0);
    take_sum += grow;
    if (served && grow > 0) granted = take_sum;
  }
  const uint64_t takers = __builtin_amdgcn_ballot_w64(granted > 0);
  if (lane == 0) wave_granted[wave] = 0;
  if (takers != 0 && lane == 63 - __builtin_clzll(takers)) wave_granted[wave] = granted;
  if (tid == 0) back_at[p.B] = all_back;
  __syncthreads();
  granted = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) granted = max(granted, wave_granted[w]);

  // the block given back u-th, and the one taken j-th
  auto given = [&](int u) {
    const int b = last_not_above(back_at, p.B, u);
    return p.table[static_cast<int64_t>(b) * p.table_ld + min(row_want[b] + u - back_at[b], p.table_ld - 1)];
  };
  auto taken = [&](int j) {
    const int s = max(top - 1 - j, 0);
    return s < n_free ? p.free[s] : given(s - n_free);
  };
  if (what & kCells) {
    for (int64_t u = first; u < all_back && u < p.n_blocks - n_free; u += step) p.free[n_free + u] = given(static_cast<int>(u));
    for (int64_t j = first; j < granted; j += step) {
      const int b = last_not_above(take_at, p.B, static_cast<int>(j));
      p.table[static_cast<int64_t>(b) * p.table_ld + row_have[b] + static_cast<int>(j) - take_at[b]] = taken(static_cast<int>(j));
    }
    for (int64_t i = first; i < n_slots; i += step) {
      const int b = static_cast<int>(i / p.T), t = static_cast<int>(i - static_cast<int64_t>(b) * p.T);
      int32_t slot = -1;
      if (t < row_new[b]) {
        const int64_t pos = static_cast<int64_t>(row_len[b]) + t;
        const int c = static_cast<int>(pos >> p.lg), old = row_have[b];
        const int32_t block = c >= old ? taken(take_at[b] + c - old)
                              : i == first ? first_block
                                           : p.table[static_cast<int64_t>(b) * p.table_ld + c];
        slot = static_cast<int32_t>((static_cast<uint32_t>(block) << p.lg) + static_cast<uint32_t>(pos & ((1 << p.lg) - 1)));
      }
      p.slots[i] = slot;
    }
  }
  if ((what & kState) && blockIdx.x == 0) {
    __syncthreads();  // one workgroup may write over what it has read
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (PER * tid + k < p.B) p.held_out[PER * tid + k] = want[k];
    if (tid == 0) p.n_free_out[0] = top - granted;
  }
}

// ------------------------------------------------------------ attn_rope

struct RopeParams {
  const uint16_t* qg;  // [B, T, Hq, q_head] (token stride qg_ld), q first in each head
  const uint16_t* kn;  // [B, T, Hkv, D] (token stride kv_ld)
  const uint16_t* vn;
  int64_t qg_ld, kv_ld;
  const void* qw;  // [D] norm weights, or both null: no norm
  const void* kw;
  int wdt;
  const int32_t* pos0;    // [B] position of each row's first token
  const int32_t* slots;   // [B, T] slot of each token, < 0: padding; or null: row b's own block
  const uint64_t* turns;  // [rot / 2] turns of a pair per position, as a fraction of 2^64
  uint16_t* q;            // [B, T, Hq, D]
  uint16_t* keys;         // [n_blocks, Hkv, block, D]
  uint16_t* values;
  int B, T, Hq, Hkv, q_head, block, rot;
  int64_t n_slots;  // n_blocks * block
  float eps, factor;
  uint32_t per_tok;  // waves of a token: q_items + 2 kv_items
  int q_items, kv_items;
};

// y = x / sqrt(mean(x^2) + eps) * w, its pairs turned by pos * turns[i] (a turn
// is 2 pi) and stretched by factor; everything in fp32, rounded once.  With r the
// norm's factor, each dim is y = r (A x + B x'), x' the other of its pair, A = w
// cos and B = -+ w' sin: A and B serve every head of a token.  A dim that does not
// turn takes x' = 0, not B = 0 alone: 0 times an inf or NaN beside it is NaN.
// A wave takes NU groups of 512 / D heads of one token and one kind (q, k or v),
// 8 dims a lane, x' by a load of its own (from the L1).  The angles are formed by
// one lane a dim and handed round in LDS; they are exact at any position: pos *
// turns in 64-bit integers drops whole turns by itself, where pos * frequency in
// fp32 is off by 0.06 rad at a million, and its top 32 bits go to the hardware's
// sine and cosine, which take turns.
// Bound by memory and arithmetic together for many tokens (4096 tokens of 16 + 2 x
// 4 heads of 256, 100 MB from a cold cache: 24.8 us, their plain copy 19; with 4
// dims a lane, x' by a lane shuffle, each wave's angles by the lanes that use them
// and a select per dim 35), by the launch and a few latencies for few (64 tokens
// 3.6).  One / two / four / eight groups a wave, us: 340 tokens 5.0 / - / 5.5 / -;
// 680 14.2 / 6.7 / 7.5 / 9.4; 4096 70 / 24.8 / 26.4 / 39.3.
constexpr int kRopeGroups = 2;      // groups of a wave
constexpr int64_t kRopeFew = 8192;  // heads of all tokens up to which a wave takes one
template <int D, int NU, bool IL>
__global__ __launch_bounds__(256) void attn_rope_kernel(const RopeParams p) {
  constexpr int LPH = D / 8, HPU = 64 / LPH;  // lanes per head, heads per group
  typedef typename RowVec<8>::type vec;
  __shared__ __align__(16) float trig[4][2][D];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t bt = (blockIdx.x * 4u + wave) / p.per_tok;
  if (bt >= static_cast<uint32_t>(p.B) * p.T) return;  // wave-uniform
  int item = static_cast<int>(blockIdx.x * 4u + wave - bt * p.per_tok);
  // q's, k's, then v's groups
  const bool is_q = item < p.q_items, is_k = !is_q && item < p.q_items + p.kv_items;
  if (!is_q) item -= is_k ? p.q_items : p.q_items + p.kv_items;
  const int H = is_q ? p.Hq : p.Hkv;
  const int b = static_cast<int>(bt / p.T), t = static_cast<int>(bt - static_cast<uint32_t>(b) * p.T);
  const int h0 = item * NU * HPU + lane / LPH, d0 = lane % LPH * 8;  // heads h0, h0 + HPU, ..

  const uint16_t* src = is_q ? p.qg + bt * p.qg_ld : (is_k ? p.kn : p.vn) + bt * p.kv_ld;
  const int head_ld = is_q ? p.q_head : D;
  const int half = p.rot / 2;
  const bool turned = d0 < p.rot && (is_q || is_k), lower = d0 < half;
  const bool whole = half % 8 == 0;  // a lane's 8 dims have their partners in one other lane's
  vec raw[NU], other[NU];
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    const uint16_t* row = src + min(h0 + n * HPU, H - 1) * head_ld;
    raw[n] = *reinterpret_cast<const vec*>(row + d0);
    other[n] = vec{};
    if (!IL && turned) {
      if (whole) {
        other[n] = *reinterpret_cast<const vec*>(row + (lower ? d0 + half : d0 - half));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = d0 + e;
          const uint16_t x = row[d < half ? d + half : d < p.rot ? d - half : d];
          other[n][e] = d < p.rot ? x : 0;
        }
      }
    }
  }
  // where k and v go: row `at` of block `page`
  uint32_t pos, page, at;
  bool pad = false;
  if (p.slots != nullptr) {
    const int32_t slot = p.slots[bt];
    pad = slot < 0 || slot >= p.n_slots;
    page = pad ? 0 : static_cast<uint32_t>(slot) / static_cast<uint32_t>(p.block);
    at = static_cast<uint32_t>(slot) - page * p.block;
    pos = static_cast<uint32_t>(max(p.pos0[b], 0)) + t;
  } else {
    page = b;
    at = pos = static_cast<uint32_t>(first_pos(p.pos0, b, p.T, p.block)) + t;
  }
  uint16_t* dst = is_q ? p.q + static_cast<int64_t>(bt) * p.Hq * D
                       : (is_k ? p.keys : p.values) + (static_cast<int64_t>(page) * p.Hkv * p.block + at) * D;
  const int64_t dst_ld = is_q ? D : static_cast<int64_t>(p.block) * D;
  if (!is_q && pad) return;
  if (!is_q && !is_k) {  // v goes into its slot as is
#pragma unroll
    for (int n = 0; n < NU; ++n)
      if (h0 + n * HPU < H) *reinterpret_cast<vec*>(dst + (h0 + n * HPU) * dst_ld + d0) = raw[n];
    return;
  }

  // the weights of the lane's dims and of their partners
  const void* w = is_q ? p.qw : p.kw;
  float A[8], B[8];
  auto load_w = [&](int i, float* out) {
    if (w == nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = 1.0f;
    } else if (p.wdt == GDN_DTYPE_F32) {
      typedef float w8 __attribute__((ext_vector_type(8), aligned(4)));
      const w8 v = *reinterpret_cast<const w8*>(static_cast<const float*>(w) + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = v[e];
    } else {
      const vec v = *reinterpret_cast<const vec*>(static_cast<const uint16_t*>(w) + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = p.wdt == GDN_DTYPE_BF16 ? bf16_to_f32(v[e]) : f16_to_f32(v[e]);
    }
  };
  load_w(d0, A);
  if constexpr (IL) {
#pragma unroll
    for (int e = 0; e < 8; ++e) B[e] = A[e ^ 1];
  } else {
    load_w(!turned || !whole ? d0 : lower ? d0 + half : d0 - half, B);
    if (turned && !whole) {
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        float one[8];
        load_w(min(d < half ? d + half : d < p.rot ? d - half : d, D - 8), one);
        const int skip = max((d < half ? d + half : d < p.rot ? d - half : d) - (D - 8), 0);
        float v = one[0];
#pragma unroll
        for (int k = 1; k < 8; ++k) v = k == skip ? one[k] : v;
#pragma unroll
        for (int k = 0; k < 8; ++k) B[k] = k == e ? v : B[k];
      }
    }
  }
  // cosine and signed sine of dim d < rot (to the last turned lane's end)
  float* cs = trig[wave][0];
  float* sn = trig[wave][1];
  for (int d = lane; d < ((p.rot + 7) & ~7); d += 64) {
    float c = 1.0f, s = 0.0f;
    if (d < p.rot) {
      const uint64_t f = p.turns[IL ? d / 2 : d < half ? d : d - half];
      const uint32_t phase = static_cast<uint32_t>(f >> 32) * pos + __umulhi(static_cast<uint32_t>(f), pos);
      const float x = static_cast<float>(static_cast<int32_t>(phase)) * 0x1p-32f;
      c = __builtin_amdgcn_cosf(x) * p.factor;
      s = __builtin_amdgcn_sinf(x) * p.factor;
      if (IL ? d % 2 == 0 : d < half) s = -s;
    }
    cs[d] = c;
    sn[d] = s;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  {
    const int d = turned ? d0 : 0;
    const f32x4 c0 = *reinterpret_cast<const f32x4*>(cs + d), c1 = *reinterpret_cast<const f32x4*>(cs + d + 4);
    const f32x4 s0 = *reinterpret_cast<const f32x4*>(sn + d), s1 = *reinterpret_cast<const f32x4*>(sn + d + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool turns = turned && d0 + e < p.rot;
      A[e] *= turns ? (e < 4 ? c0[e & 3] : c1[e & 3]) : 1.0f;
      B[e] = turns ? B[e] * (e < 4 ? s0[e & 3] : s1[e & 3]) : 0.0f;
    }
  }

#pragma unroll
  for (int n = 0; n < NU; ++n) {
    float x[8], ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = bf16_to_f32(raw[n][e]);
      ss = fmaf(x[e], x[e], ss);
    }
    float r = 1.0f;
    if (w != nullptr) {
      ss += dpp_f<GDN_DPP_QUAD_XOR1>(ss);
      ss += dpp_f<GDN_DPP_QUAD_XOR2>(ss);
      ss += dpp_f<GDN_DPP_HALF_MIRROR>(ss);
      ss += dpp_f<GDN_DPP_ROW_MIRROR>(ss);
      if constexpr (LPH == 32) {
        const auto s2 = __builtin_amdgcn_permlane16_swap(__float_as_uint(ss), __float_as_uint(ss), false, false);
        ss = __uint_as_float(s2[0]) + __uint_as_float(s2[1]);
      }
      r = rsqrtf(ss / D + p.eps);
    }
    typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));
    words out;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const bool turns = d0 + e < p.rot;  // (both of a pair, as rot is even)
      const float o0 = IL ? (turns ? x[e + 1] : 0.0f) : bf16_to_f32(other[n][e]);
      const float o1 = IL ? (turns ? x[e] : 0.0f) : bf16_to_f32(other[n][e + 1]);
      out[e / 2] = pk_bf16(r * fmaf(A[e], x[e], B[e] * o0), r * fmaf(A[e + 1], x[e + 1], B[e + 1] * o1));
    }
    if (h0 + n * HPU < H) *reinterpret_cast<words*>(dst + (h0 + n * HPU) * dst_ld + d0) = pad ? words{0u, 0u, 0u, 0u} : out;
  }
}

int lg2(int64_t x) {  // of a power of two, else -1
  return x > 0 && (x & (x - 1)) == 0 ? __builtin_ctzll(static_cast<uint64_t>(x)) : -1;
}

// ------------------------------------------------------------ attention

// One launch covers a step: the workgroups of the shared prefix first (all rows
// of the batch, read once per row tile), then each row's own keys.
struct StepParams : PagedParams {
  int n_prefix, n_own;        // key ranges
  int len_prefix, len_own;    // keys of a range
  int prefix_tiles, own_tiles;  // row tiles
  int prefix_few, own_few;      // of the 16 rows of attn_rows, not the PR of attn_tile
};

// Rows 16 rb .. of kv-head hkv (of batch entry b, or of the whole batch) over key
// range `split`, by W waves.  Every wave takes 16 KT keys of a step of 16 KT W and
// keeps a softmax state of its own; nothing in the loop waits for another wave.
// K and V go to the wave's own 16 KB of LDS by direct loads of whole rows (K as
// fragments from memory, 64 bytes of a row at a time, took 1.6 times as long from
// a warm cache), their 16-byte granules swizzled on the way: K's by (key & 15), so
// that 16-byte fragment reads of 16 keys hit distinct banks, V's by 2 (key & 7), so
// that its transposed reads of 4 x 4 keys do.  K of the next step is asked for as
// soon as this one's scores are formed, V as soon as its products are: a CU has up
// to 128 KB in flight.  Bound by memory: a full cache of 64 rows of 4096 keys at 4
// kv-heads of 256 (1.07 GB) takes 164 us, 6.6 TB/s (without the hint that the keys
// are read once 186).
// More than 16 rows may take several workgroups, each of which reads the keys: from
// the L2, as those of one range run on one XCD.  Tiles of 32 rows in the same way
// (O and Q in 192 registers) were within 10% of attn_tile either way at 17 to 32
// rows and slower beyond.
template <int D, int W>
constexpr int rows_lds() {
  constexpr int kv = W * 2 * 256 * 16 * 2, merge = W * 16 * D * 4 + 2 * W * 16 * 4;
  return kv > merge ? kv : merge;
}
template <int D, int W>
__device__ __forceinline__ void attn_rows(const PagedParams& p, unsigned char* smem, int b, int hkv, int rb, int split) {
  constexpr int KT = 256 / D;         // 16-key tiles per wave and step
  constexpr int KW = 16 * KT;         // keys per wave and step
  constexpr int KS = KW * W;          // keys per step
  constexpr int NS = D / 32, NJ = D / 16;
  constexpr int KROW = D / 8;         // 16-byte granules per row
  constexpr int LD = KW * KROW / 64;  // direct loads of 1 KB per wave, step and operand
  constexpr int STAGE = KW * D * 2;   // bytes
  const int g = p.Hq / p.Hkv;
  const int row0 = 16 * rb, n_rows = min(tile_rows(p, g) - row0, 16);  // this workgroup's
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lq = lane >> 4;
  const int tokens = row_tokens(p, b);
  const int p0 = row_start(p, b, tokens);
  const KeyRange range = key_range(p, split, p0, min((row0 + 15) / g, tokens - 1), row0 / g < tokens);
  const int k_lo = range.lo + KW * wave, k_hi = range.hi;  // this wave's keys: KW from k_lo, k_lo + KS, ..
  const int k_free = prefix_of(p) ? k_hi : min(p0 + row0 / g + 1, k_hi);  // keys below this are visible to every row
  const int n_step = k_hi > k_lo ? (k_hi - k_lo + KS - 1) / KS : 0;

  // lane l holds the block of the wave's step page0 + l
  int page0 = 0, pages = 0;
  auto load_pages = [&](int i) {
    page0 = i;
    pages = block_of(p, b, min(k_lo + KS * (i + lane), k_hi - 1));
  };
  // the wave's keys of step i: rows past the range read as zeros
  unsigned char* ks = smem + wave * (2 * STAGE);
  const unsigned char* vs = ks + STAGE;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ks)));
  const int key0 = lane / KROW, gran = lane % KROW;
  static_assert(64 % KROW == 0, "whole rows per load");
  constexpr int RL = 64 / KROW;  // rows per load
  // one row tile's own keys are read by one workgroup, where none of them are shared
  const bool once = !prefix_of(p) && p.pos_min == p.key0 && tile_rows(p, g) <= 16;
  auto load = [&](const uint16_t* pool, int i, uint32_t lds, int twist) {
    const int kb = k_lo + KS * i;
    const int64_t off = key_off<D>(p, b, hkv, kb, __builtin_amdgcn_readlane(pages, i - page0)) * 2;
    const u32x4 rsrc = buf_words(reinterpret_cast<const unsigned char*>(pool) + off, min(k_hi - kb, KW) * (D * 2));
#pragma unroll
    for (int c = 0; c < LD; ++c) {
      const int row = c * RL + key0;
      const uint32_t off = row * (D * 2) + (gran ^ (twist == 1 ? row & 15 : 2 * (row & 7))) * 16;
      if (once) lds_dma16_once(rsrc, off, lds + c * 1024);
      else lds_dma16(rsrc, off, lds + c * 1024);
    }
  };

  if (n_step > 0) {
    load_pages(0);
    load(p.kc, 0, lds0, 1);
  }
  // lane lr's row: Q as the B operand of S^T = K Q^T
  const RowAt at = row_at(p, b, hkv, g, row0 + (lr < n_rows ? lr : 0));
  const bool row_ok = lr < n_rows && (prefix_of(p) || at.t < tokens);
  const int kmax = prefix_of(p) ? INT_MAX : p0 + at.t;  // last key the row may see
  u32x4 qr[NS];
  {
    const uint16_t* qrow = p.q + ((static_cast<int64_t>(at.b) * p.T + at.t) * p.Hq + at.hq) * D;
#pragma unroll
    for (int s = 0; s < NS; ++s) qr[s] = *reinterpret_cast<const u32x4*>(qrow + 32 * s + 8 * lq);
  }
  if (n_step > 0) load(p.vc, 0, lds0 + STAGE, 2);
  bf16x8 qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) qf[s] = __builtin_bit_cast(bf16x8, row_ok ? qr[s] : u32x4{0u, 0u, 0u, 0u});

  float m = -FLT_MAX, l = 0.0f;  // running max (log2 units) and this lane's share of the sum
  f32x4 o[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < n_step; ++i) {
    const int kb = k_lo + KS * i;
    const bool more = i + 1 < n_step;
    if (more && i + 1 - page0 >= 64) load_pages(i + 1);
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LD) : "memory");  // K is there, V may be on its way
    // S^T = K Q^T: lane (r, q) holds keys 16 kt + 4 q + e of row r
    f32x4 sc[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < NS; ++s)
        a = mfma16(*reinterpret_cast<const bf16x8*>(ks + (16 * kt + lr) * (D * 2) + ((4 * s + lq) ^ lr) * 16), qf[s], a);
      sc[kt] = a;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // K is read
    if (more) load(p.kc, i + 1, lds0, 1);

    if (kb + KW > k_free) {  // some row does not see them all
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = kb + 16 * kt + 4 * lq + e;
          if (!(key <= kmax && key < k_hi)) sc[kt][e] = -INFINITY;
        }
    }
    float mb = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) mb = fmaxf(mb, sc[kt][e]);
    mb = rows_max(mb) * p.scale_log2;
    // the max is raised only when a row's grows by more than 8 (P stays below 2^8): most steps rescale nothing
    if (__builtin_amdgcn_ballot_w64(mb > m + 8.0f) != 0) {
      const float m_new = fmaxf(m, mb);
      const float alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int j = 0; j < NJ; ++j) o[j] *= alpha;
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[kt][e] = __builtin_amdgcn_exp2f(fmaf(sc[kt][e], p.scale_log2, -m));
        l += sc[kt][e];
      }
    if (more) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LD) : "memory");  // V is there, the next K on its way
    else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    // O^T += V^T P^T: P (as bf16) in the accumulators' own lanes, V^T by transposed LDS reads of
    // keys 4 q .. 4 q + 3 (lane r: key 4 q + r / 4, dims 16 j + 4 (r % 4) ..)
    const int key = 4 * lq + (lr >> 2);
    const unsigned char* va = vs + key * (D * 2) + 16 * ((lr & 3) >> 1) + 8 * (lr & 1);
    const int twist = 32 * (key & 7);
    auto v_read = [&](int j, int kt) {
      return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(va + kt * 16 * (D * 2) + ((32 * j) ^ twist)));
    };
    if constexpr (KT == 1) {
      const i16x4 pb = __builtin_bit_cast(i16x4, u32x2{pk_bf16(sc[0][0], sc[0][1]), pk_bf16(sc[0][2], sc[0][3])});
#pragma unroll
      for (int j = 0; j < NJ; ++j) o[j] = mfma16k16(v_read(j, 0), pb, o[j]);
    } else {
      const bf16x8 pb = __builtin_bit_cast(bf16x8, u32x4{pk_bf16(sc[0][0], sc[0][1]), pk_bf16(sc[0][2], sc[0][3]),
                                                         pk_bf16(sc[1][0], sc[1][1]), pk_bf16(sc[1][2], sc[1][3])});
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        o[j] = mfma16(__builtin_bit_cast(bf16x8, i16x8(__builtin_shufflevector(v_read(j, 0), v_read(j, 1), 0, 1, 2, 3, 4, 5, 6, 7))),
                      pb, o[j]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // V is read
    if (more) load(p.vc, i + 1, lds0 + STAGE, 2);
  }
  l = rows_sum(l);

  // the waves' states merge: thread (row, column piece)
  __syncthreads();
  // [W][16][D], a row's 16-byte granules XOR-swizzled by the row: unswizzled, the accumulators' 16 rows lie in the
  // same banks, and the merge took 4.2 us, not 1.1
  f32x4* Os = reinterpret_cast<f32x4*>(smem);
  float* Ms = reinterpret_cast<float*>(smem) + W * 16 * D;  // [W][16]
  float* Ls = Ms + W * 16;
#pragma unroll
  for (int j = 0; j < NJ; ++j) Os[(wave * 16 + lr) * (D / 4) + ((4 * j + lq) ^ lr)] = o[j];
  if (lq == 0) {
    Ms[wave * 16 + lr] = m;
    Ls[wave * 16 + lr] = l;
  }
  __syncthreads();
  constexpr int CW = D / (4 * W);  // columns per thread, in pieces of 4, 16 W apart
  static_assert(CW % 4 == 0, "whole pieces");
  const int mr = threadIdx.x / (4 * W), c0 = (threadIdx.x % (4 * W)) * 4;
  if (mr >= n_rows) return;
  const RowAt mat = row_at(p, b, hkv, g, row0 + mr);
  if (!prefix_of(p) && mat.t >= tokens) {  // a padded token
    if (p.n_split == 1) {
#pragma unroll
      for (int c = 0; c < CW / 4; ++c) store_zero4<D>(p, mat.b, mat.t, mat.hq, c0 + 16 * W * c);
    }
    return;
  }
  float ms = -FLT_MAX, mw[W], ls = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) ms = fmaxf(ms, Ms[w * 16 + mr]);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    mw[w] = __builtin_amdgcn_exp2f(Ms[w * 16 + mr] - ms);
    ls += mw[w] * Ls[w * 16 + mr];
  }
  f32x4 acc[CW / 4];
#pragma unroll
  for (int c = 0; c < CW / 4; ++c) {
    acc[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W; ++w)
      acc[c] += mw[w] * Os[(w * 16 + mr) * (D / 4) + ((c0 / 4 + 4 * W * c) ^ mr)];
  }
  if (p.n_split == 1) {
    store_row<D, CW / 4, 16 * W>(p, (mat.b * p.T + mat.t) * p.Hq + mat.hq, c0, acc, ls);
    return;
  }
  const int64_t pr = part_row(p, mat.b, hkv, mat.row) + split_at(p, split);
#pragma unroll
  for (int c = 0; c < CW / 4; ++c) *reinterpret_cast<f32x4*>(p.part + pr * D + c0 + 16 * W * c) = acc[c];
  if (c0 == 0) {
    const int64_t n_part = static_cast<int64_t>(p.B) * p.Hkv * p.rows_pad * p.n_split;
    p.part[n_part * D + pr] = ms;
    p.part[n_part * (D + 1) + pr] = ls;
  }
}

template <int D>
constexpr int step_threads() { return D == 256 ? 512 : 256; }

template <int D>
__global__ __launch_bounds__(step_threads<D>()) void attn_step_kernel(const StepParams p) {
  constexpr int KG = D == 256 ? 2 : 1, W = step_threads<D>() / 64;
  constexpr int kTile = tile_lds<D, KG, PagedParams>(), kRows = rows_lds<D, W>();
  __shared__ __align__(128) unsigned char smem[kTile > kRows ? kTile : kRows];
  // (kv-head, range) pairs run fastest, so that the row tiles that read a range's keys run on one XCD where
  // the pairs are a multiple of the eight, and its L2 reads them once
  PagedParams r = p;
  int i = blockIdx.x;
  const int n_prefix = p.Hkv * p.n_prefix * p.prefix_tiles;
  r.prefix = i < n_prefix;
  if (!r.prefix) i -= n_prefix;
  r.split0 = r.prefix ? 0 : p.n_prefix;
  r.split_len = r.prefix ? p.len_prefix : p.len_own;
  const int tiles = r.prefix ? p.prefix_tiles : p.own_tiles;
  const int pairs = p.Hkv * (r.prefix ? p.n_prefix : p.n_own);
  const int tb = i / pairs, hs = i - tb * pairs;
  const int split = hs / p.Hkv, hkv = hs - split * p.Hkv;
  const int batch = r.prefix ? 1 : p.B;
  const int tile = tb / batch, b = tb - tile * batch;
  if (r.prefix ? p.prefix_few : p.own_few) attn_rows<D, W>(r, smem, b, hkv, tiles - 1 - tile, split);
  else attn_tile<D, KG>(r, smem, b, hkv, tiles - 1 - tile, split);  // longest key ranges first
}

// One wave per (token, q-head): its ranges' partial results merged, as
// attn_combine_kernel does, and a padded token's zeros.  The first NB ranges'
// sums, the gate and all maxima are loaded before any is used: the launch is a
// few memory latencies long.  A range without a key of the row (l = 0) may not
// have written its sums: they are loaded all the same and dropped.
template <int D>
__global__ __launch_bounds__(256) void step_combine_kernel(const PagedParams p) {
  constexpr int EPL = D / 64, NB = 8;
  typedef float vec __attribute__((ext_vector_type(EPL)));
  typedef uint16_t hvec __attribute__((ext_vector_type(EPL)));
  const int lane = threadIdx.x & 63;
  const int item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int g = p.Hq / p.Hkv;
  const int bt = item / p.Hq, hq = item - bt * p.Hq;
  const int b = bt / p.T, t = bt - b * p.T;
  if (b >= p.B) return;
  const int64_t n_part = static_cast<int64_t>(p.B) * p.Hkv * p.rows_pad * p.n_split;
  const int64_t pr = part_row(p, b, hq / g, t * g + hq % g);
  const float* pm = p.part + n_part * D + pr;
  const float* pl = p.part + n_part * (D + 1) + pr;
  uint16_t* out = p.out + (static_cast<int64_t>(bt) * p.Hq + hq) * D + EPL * lane;
  hvec gate = {};
  if (p.qg != nullptr) gate = *reinterpret_cast<const hvec*>(p.qg + bt * p.qg_ld + hq * 2 * D + D + EPL * lane);
  const int tokens = row_tokens(p, b);
  vec acc = {}, v[NB];
  float m = -FLT_MAX, lsum = 0.0f;
  for (int s0 = 0; s0 < p.n_split; s0 += 64) {
    const int n = min(64, p.n_split - s0);
    const float ls = pl[s0 + min(lane, n - 1)], ms = pm[s0 + min(lane, n - 1)];
    auto load = [&](int s) {
#pragma unroll
      for (int i = 0; i < NB; ++i)
        v[i] = *reinterpret_cast<const vec*>(p.part + (pr + s0 + min(s + i, n - 1)) * D + EPL * lane);
    };
    load(0);
    const bool has = lane < n && ls != 0.0f;
    const float m_new = fmaxf(m, wave_max(has ? ms : -FLT_MAX));
    const float keep = __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    const float w = has ? __builtin_amdgcn_exp2f(ms - m) : 0.0f;  // the lane's range
    acc *= keep;
    lsum = lsum * keep + wave_sum(has ? w * ls : 0.0f);
    for (int s = 0; s < n; s += NB) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const float wi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), min(s + i, 63)));
        if (s + i < n && wi != 0.0f) acc += wi * v[i];  // wave-uniform
      }
      if (s + NB < n) load(s + NB);
    }
  }
  const float inv_l = 1.0f / lsum;  // (0: every score is -inf, whose softmax is NaN)
  hvec y;
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    float x = lsum == 0.0f ? __builtin_nanf("") : acc[e] * inv_l;
    if (p.qg != nullptr) x *= sigmoid(bf16_to_f32(gate[e]));
    y[e] = f32_to_bf16(x);
  }
  *reinterpret_cast<hvec*>(out) = t < tokens ? y : hvec{};
}

}  // namespace

extern "C" int gdn_paged_tables(const int32_t* lengths, const int32_t* n_new, int32_t* table, int64_t table_ld,
                                const int32_t* held, int32_t* free_blocks, const int32_t* n_free, int32_t* held_out,
                                int32_t* n_free_out, int32_t* slots, int64_t B, int64_t T, int64_t block,
                                int64_t shared, int64_t n_blocks, void* stream) {
  using gdn_host::fail;
  const int lg = lg2(block);
  if (B < 0 || T < 0 || lg < 0 || lg > 20 || table_ld < 0 || table_ld > INT32_MAX || n_blocks < 0 || shared < 0 ||
      shared > table_ld)
    return fail(GDN_ERR_INVALID, "gdn_paged_tables: bad sizes (blocks are powers of two up to 2^20; shared <= table width)");
  if (B > kTableRows) return fail(GDN_ERR_UNSUPPORTED, "gdn_paged_tables: at most %d rows (got %lld)", kTableRows, (long long)B);
  if (B * T > INT32_MAX || n_blocks * block > INT32_MAX || B * table_ld > INT32_MAX)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_paged_tables: tokens, slots and table entries must each be below 2^31");
  if (B == 0) {
    if (n_free_out != n_free) return fail(GDN_ERR_INVALID, "gdn_paged_tables: no rows");
    return GDN_OK;
  }
  if (!lengths || (table_ld > 0 && !table) || !held || (n_blocks > 0 && !free_blocks) || !n_free || !held_out ||
      !n_free_out || (T > 0 && !slots))
    return fail(GDN_ERR_INVALID, "gdn_paged_tables: null pointer");
  const TableParams p = {lengths, n_new, table, held, free_blocks, n_free, held_out, n_free_out, slots,
                         static_cast<int>(B), static_cast<int>(T), static_cast<int>(table_ld), lg,
                         static_cast<int>(shared), static_cast<int>(n_blocks)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  // a few tokens a thread: more would wait for each other's loads, fewer repeat the sums
  const int64_t groups = (B * T + 4 * kTableThreads - 1) / (4 * kTableThreads);
  const unsigned grid = static_cast<unsigned>(groups < 1 ? 1 : groups > 512 ? 512 : groups);
  const bool behind = grid > 1 && (held_out == held || n_free_out == n_free);
  auto launch = [&](unsigned n, int what) {
    if (B <= kTableThreads) hipLaunchKernelGGL(tables_kernel<1>, dim3(n), dim3(kTableThreads), 0, st, p, what);
    else hipLaunchKernelGGL(tables_kernel<kTableRows / kTableThreads>, dim3(n), dim3(kTableThreads), 0, st, p, what);
    return gdn_host::check_launch("gdn_paged_tables");
  };
  const int rc = launch(grid, behind ? kCells : kCells | kState);
  return rc != GDN_OK || !behind ? rc : launch(1, kState);
}

extern "C" int gdn_attn_rope(const void* qg, int64_t qg_ld, int64_t q_head, const void* k_new, const void* v_new,
                             int64_t kv_ld, const void* q_norm_w, const void* k_norm_w, int w_dtype, float eps,
                             const int32_t* pos0, const int32_t* slots, const uint64_t* turns, float factor,
                             int interleaved, void* q_out, void* keys, void* values, int64_t B, int64_t T, int64_t Hq,
                             int64_t Hkv, int64_t D, int64_t n_blocks, int64_t block, int64_t rot, void* stream) {
  using gdn_host::fail;
  if (D != 128 && D != 256) return fail(GDN_ERR_UNSUPPORTED, "gdn_attn_rope: head dim must be 128 or 256 (got %lld)", (long long)D);
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || q_head < D || n_blocks < 0 || block <= 0 ||
      block > INT32_MAX || (!slots && (n_blocks != B || block < T)))
    return fail(GDN_ERR_INVALID, "gdn_attn_rope: bad sizes");
  if (rot < 0 || rot > D || rot % 2 != 0)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_attn_rope: rotary dims %lld not supported for head dim %lld", (long long)rot,
                (long long)D);
  if ((q_norm_w == nullptr) != (k_norm_w == nullptr) || (q_norm_w && !gdn_host::dtype_ok(w_dtype)) || !(eps >= 0.0f))
    return fail(GDN_ERR_INVALID, "gdn_attn_rope: bad norm weights or eps");
  if (B * T == 0) return GDN_OK;
  if (!qg || !k_new || !v_new || !pos0 || (rot > 0 && !turns) || !q_out || !keys || !values)
    return fail(GDN_ERR_INVALID, "gdn_attn_rope: null pointer");
  if (B * T * (Hq + 2 * Hkv) > INT32_MAX || Hq * q_head > INT32_MAX)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_attn_rope: problem too large");
  if (slots && n_blocks * block > INT32_MAX)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_attn_rope: slots must be below 2^31");
  if (qg_ld == 0) qg_ld = q_head * Hq;
  if (kv_ld == 0) kv_ld = Hkv * D;
  if (qg_ld < q_head * (Hq - 1) + D || kv_ld < Hkv * D)
    return fail(GDN_ERR_INVALID, "gdn_attn_rope: token strides below the rows");
  RopeParams p;
  p.qg = static_cast<const uint16_t*>(qg);
  p.kn = static_cast<const uint16_t*>(k_new);
  p.vn = static_cast<const uint16_t*>(v_new);
  p.qg_ld = qg_ld;
  p.kv_ld = kv_ld;
  p.qw = q_norm_w;
  p.kw = k_norm_w;
  p.wdt = w_dtype;
  p.pos0 = pos0;
  p.slots = slots;
  p.turns = turns;
  p.q = static_cast<uint16_t*>(q_out);
  p.keys = static_cast<uint16_t*>(keys);
  p.values = static_cast<uint16_t*>(values);
  p.B = static_cast<int>(B);
  p.T = static_cast<int>(T);
  p.Hq = static_cast<int>(Hq);
  p.Hkv = static_cast<int>(Hkv);
  p.q_head = static_cast<int>(q_head);
  p.block = static_cast<int>(block);
  p.rot = static_cast<int>(rot);
  p.n_slots = n_blocks * block;
  p.eps = eps;
  p.factor = factor;
  hipStream_t st = static_cast<hipStream_t>(stream);
  // groups of heads per wave by the heads of all tokens: a wave with more runs longer, and shares its
  // angles and weights among them
  auto launch = [&](auto nu, auto il) {
    constexpr int NU = decltype(nu)::value;
    constexpr bool IL = decltype(il)::value;
    const int64_t per = NU * (512 / D);  // heads per wave
    p.q_items = static_cast<int>((Hq + per - 1) / per);
    p.kv_items = static_cast<int>((Hkv + per - 1) / per);
    p.per_tok = static_cast<uint32_t>(p.q_items + 2 * p.kv_items);
    const dim3 grid(static_cast<unsigned>((B * T * p.per_tok + 3) / 4));
    if (D == 256) hipLaunchKernelGGL((attn_rope_kernel<256, NU, IL>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((attn_rope_kernel<128, NU, IL>), grid, dim3(256), 0, st, p);
  };
  auto groups_per_wave = [&](auto il) {
    const int64_t rows = B * T * (Hq + 2 * Hkv);
    if (rows <= kRopeFew) launch(std::integral_constant<int, 1>{}, il);
    else launch(std::integral_constant<int, kRopeGroups>{}, il);
  };
  if (interleaved) groups_per_wave(std::true_type{});
  else groups_per_wave(std::false_type{});
  return gdn_host::check_launch("gdn_attn_rope");
}

extern "C" size_t gdn_paged_attn_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                                 int64_t n_ranges) {
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || n_ranges <= 1) return 0;
  return static_cast<size_t>(B * T * Hq * n_ranges) * (D + 2) * sizeof(float);
}

extern "C" int gdn_paged_attn(const void* q, const void* qg, int64_t qg_ld, const void* keys, const void* values,
                              const int32_t* table, int64_t table_ld, const int32_t* pos0, const int32_t* n_new,
                              void* out, float scale, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                              int64_t n_blocks, int64_t block, int64_t kv_len_max, int64_t shared, int64_t n_prefix,
                              int64_t n_own, int64_t prefix_rows, int64_t own_rows, void* workspace,
                              size_t workspace_bytes, void* stream) {
  using gdn_host::fail;
  if (D != 128 && D != 256) return fail(GDN_ERR_UNSUPPORTED, "gdn_paged_attn: head dim must be 128 or 256 (got %lld)", (long long)D);
  const int lg = lg2(block);
  if (lg < 6 || lg > 20)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_paged_attn: blocks must be powers of two from 64 to 2^20 keys (got %lld)", (long long)block);
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || n_blocks <= 0 || n_blocks > INT32_MAX ||
      table_ld <= 0 || table_ld > INT32_MAX || table_ld * block > INT32_MAX ||
      kv_len_max > table_ld * block || shared < 0 || shared > table_ld ||
      kv_len_max < shared * block + (n_new ? 0 : T) || n_prefix < 0 || n_prefix > 65535 || n_own < 1 ||
      n_own > 65535 || (n_prefix > 0 && shared == 0) || (prefix_rows != 16 && prefix_rows != PR) ||
      (own_rows != 16 && own_rows != PR))
    return fail(GDN_ERR_INVALID,
                "gdn_paged_attn: bad sizes (kv_len_max must lie in [shared * block + T, table width * block])");
  if (!(scale > 0.0f)) return fail(GDN_ERR_INVALID, "gdn_paged_attn: scale must be positive");
  if (B * T == 0) return GDN_OK;
  if (!q || !keys || !values || !table || !pos0 || !out) return fail(GDN_ERR_INVALID, "gdn_paged_attn: null pointer");
  if (qg_ld == 0) qg_ld = 2 * Hq * D;
  if (qg && qg_ld < 2 * Hq * D) return fail(GDN_ERR_INVALID, "gdn_paged_attn: gate token stride below the row");
  if (!gdn_host::aligned(q, 16) || !gdn_host::aligned(keys, 16) || !gdn_host::aligned(values, 16) ||
      !gdn_host::aligned(out, 8) || (qg && (!gdn_host::aligned(qg, 8) || qg_ld % 4 != 0)))
    return fail(GDN_ERR_INVALID, "gdn_paged_attn: misaligned pointer");
  const int64_t g = Hq / Hkv, rows = T * g, n_split = n_prefix + n_own;
  // (ranges of up to 65535 are rounded up to steps, and asked for a step of all lanes ahead: 2^30 keys leave room)
  if (table_ld * block > (int64_t(1) << 30) || Hkv > 16384 || B > 65535 || B * T * Hq > INT32_MAX / 2 || Hkv * n_split > INT32_MAX ||
      B * Hkv * rows * n_split * (D + 2) > (int64_t(1) << 40))
    return fail(GDN_ERR_UNSUPPORTED, "gdn_paged_attn: problem too large");
  const size_t need = gdn_paged_attn_workspace_bytes(B, T, Hq, Hkv, D, n_split);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !gdn_host::aligned(workspace, 16)))
    return fail(GDN_ERR_INVALID, "gdn_paged_attn: workspace of %zu bytes is below the %zu needed for %lld key ranges",
                workspace_bytes, need, (long long)n_split);
  StepParams p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.qg = static_cast<const uint16_t*>(qg);
  p.qg_ld = qg_ld;
  p.kc = static_cast<const uint16_t*>(keys);
  p.vc = static_cast<const uint16_t*>(values);
  p.pos0 = pos0;
  p.out = static_cast<uint16_t*>(out);
  p.part = static_cast<float*>(workspace);
  p.B = static_cast<int>(B);
  p.T = static_cast<int>(T);
  p.Hq = static_cast<int>(Hq);
  p.Hkv = static_cast<int>(Hkv);
  p.cap = static_cast<int>(table_ld * block);
  p.n_split = static_cast<int>(n_split);
  p.rows_pad = static_cast<int>(rows);
  p.scale_log2 = scale * kLog2e;
  p.table = table;
  p.n_new = n_new;
  p.table_ld = static_cast<int>(table_ld);
  p.lg = lg;
  p.n_blocks = static_cast<int>(n_blocks);
  hipStream_t st = static_cast<hipStream_t>(stream);
  p.key0 = static_cast<int>(n_prefix > 0 ? shared * block : 0);
  p.pos_min = static_cast<int>(shared * block);
  p.new_max = static_cast<int>(std::min(T, table_ld * block - shared * block));
  auto range_len = [](int64_t keys, int64_t n) { return static_cast<int>(((keys + n - 1) / n + KB - 1) / KB * KB); };
  p.n_prefix = static_cast<int>(n_prefix);
  p.n_own = static_cast<int>(n_own);
  p.len_prefix = n_prefix > 0 ? range_len(p.key0, n_prefix) : 0;
  p.len_own = range_len(kv_len_max - p.key0, n_own);
  auto tiles_of = [](int64_t n, int64_t tile) { return static_cast<int>((n + tile - 1) / tile); };
  p.prefix_few = prefix_rows == 16;
  p.own_few = own_rows == 16;
  p.prefix_tiles = n_prefix > 0 ? tiles_of(B * rows, prefix_rows) : 0;
  p.own_tiles = tiles_of(rows, own_rows);
  const int64_t groups = Hkv * (n_prefix * p.prefix_tiles + B * n_own * p.own_tiles);
  if (groups > INT32_MAX) return fail(GDN_ERR_UNSUPPORTED, "gdn_paged_attn: problem too large");
  if (D == 256) hipLaunchKernelGGL(attn_step_kernel<256>, dim3(static_cast<unsigned>(groups)), dim3(512), 0, st, p);
  else hipLaunchKernelGGL(attn_step_kernel<128>, dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, p);
  const int rc = gdn_host::check_launch("gdn_paged_attn");
  if (rc != GDN_OK || n_split == 1) return rc;
  const dim3 cgrid(static_cast<unsigned>((B * T * Hq + 3) / 4));
  if (D == 256) hipLaunchKernelGGL(step_combine_kernel<256>, cgrid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(step_combine_kernel<128>, cgrid, dim3(256), 0, st, p);
  return gdn_host::check_launch("gdn_paged_attn/combine");
}
