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

constexpr int kTableRows = 4096;  // rows whose running sums a workgroup keeps in LDS

__device__ __forceinline__ int32_t saturate(int64_t x) { return static_cast<int32_t>(min<int64_t>(x, INT32_MAX)); }

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

// Row b needs max(ceil((len + new) / block), shared) blocks.  Rows with more
// give the last ones back, onto the free stack's top in row order, then rows
// with fewer take from the top in row order, as far as the stack reaches: a row
// that does not get all it asks for gets none, and no row after it any.
// Every workgroup forms the running sums of all rows by itself and then takes
// its share of the cells; a cell that one writes, none reads: blocks given back
// in this call are taken from their giver's table, not from the stack.  State
// that would be written over what other workgroups read (held_out = held) is
// written by a launch of one workgroup (kState) behind the others (kCells).
constexpr int kCells = 1, kState = 2;
__global__ __launch_bounds__(256) void tables_kernel(const TableParams p, int what) {
  __shared__ int32_t back_at[kTableRows + 1], take_at[kTableRows + 1];
  __shared__ int64_t wave_back[4], wave_take[4];
  __shared__ int32_t wave_granted[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  struct Row {
    int len, n, have, back, take;
    bool fits;
  };
  auto row_of = [&](int b) {
    Row r;
    r.len = max(p.lengths[b], 0);
    r.n = p.n_new != nullptr ? min(max(p.n_new[b], 0), p.T) : p.T;
    r.have = min(max(p.held[b], 0), p.table_ld);
    const int64_t need =
        max<int64_t>((static_cast<int64_t>(r.len) + r.n + (int64_t(1) << p.lg) - 1) >> p.lg, p.shared);
    r.fits = need <= p.table_ld;
    const int want = r.fits ? static_cast<int>(need) : r.have;
    r.back = max(r.have - want, 0);
    r.take = max(want - r.have, 0);
    return r;
  };

  // running sums: thread tid has rows per * tid ..
  const int per = (p.B + 255) / 256, b0 = min(per * tid, p.B), b1 = min(b0 + per, p.B);
  int64_t back = 0, take = 0;
  for (int b = b0; b < b1; ++b) {
    const Row r = row_of(b);
    back += r.back;
    take += r.take;
  }
  int64_t back_sum = back, take_sum = take;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t x = __shfl_up(back_sum, d, 64), y = __shfl_up(take_sum, d, 64);
    if (lane >= d) {
      back_sum += x;
      take_sum += y;
    }
  }
  if (lane == 63) {
    wave_back[wave] = back_sum;
    wave_take[wave] = take_sum;
  }
  __syncthreads();
  int64_t all_back = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) {
      back_sum += wave_back[w];
      take_sum += wave_take[w];
    }
    all_back += wave_back[w];
  }
  const int n_free = min(max(p.n_free[0], 0), p.n_blocks);
  const int top = saturate(n_free + all_back);
  back = back_sum - back;
  take = take_sum - take;
  int granted = 0;
  for (int b = b0; b < b1; ++b) {
    const Row r = row_of(b);
    back_at[b] = saturate(back);
    take_at[b] = saturate(take);
    back += r.back;
    take += r.take;
    if (r.take > 0 && take <= top) granted = static_cast<int>(take);
  }
  if (tid == 0) {
    back_at[p.B] = saturate(all_back);
    take_at[p.B] = INT32_MAX;
  }
#pragma unroll
  for (int d = 32; d > 0; d /= 2) granted = max(granted, __shfl_xor(granted, d, 64));
  if (lane == 0) wave_granted[wave] = granted;
  __syncthreads();
  granted = max(max(wave_granted[0], wave_granted[1]), max(wave_granted[2], wave_granted[3]));

  // the block given back u-th, and the one taken j-th
  auto given = [&](int u) {
    const int b = last_not_above(back_at, p.B, u);
    const Row r = row_of(b);
    const int c = r.have - r.back + u - back_at[b];
    return p.table[static_cast<int64_t>(b) * p.table_ld + min(c, p.table_ld - 1)];
  };
  auto taken = [&](int j) {
    const int s = max(top - 1 - j, 0);
    return s < n_free ? p.free[s] : given(s - n_free);
  };
  auto served = [&](const Row& r, int b) { return r.fits && (r.take == 0 || take_at[b] + int64_t(r.take) <= top); };

  const int first = blockIdx.x * 256 + tid, step = gridDim.x * 256;
  if (what & kCells) {
    const int n_back = back_at[p.B];
    for (int u = first; u < n_back && u < p.n_blocks - n_free; u += step) p.free[n_free + u] = given(u);
    for (int j = first; j < granted; j += step) {
      const int b = last_not_above(take_at, p.B, j);
      p.table[static_cast<int64_t>(b) * p.table_ld + row_of(b).have + j - take_at[b]] = taken(j);
    }
    const int64_t n_slots = static_cast<int64_t>(p.B) * p.T;
    for (int64_t i = first; i < n_slots; i += step) {
      const int b = static_cast<int>(i / p.T), t = static_cast<int>(i - static_cast<int64_t>(b) * p.T);
      const Row r = row_of(b);
      int32_t slot = -1;
      if (t < r.n && served(r, b)) {
        const int64_t pos = static_cast<int64_t>(r.len) + t;
        const int c = static_cast<int>(pos >> p.lg);
        const int32_t block = c < r.have ? p.table[static_cast<int64_t>(b) * p.table_ld + c] : taken(take_at[b] + c - r.have);
        slot = static_cast<int32_t>(static_cast<uint32_t>(block) << p.lg) + static_cast<int32_t>(pos & ((1 << p.lg) - 1));
      }
      p.slots[i] = slot;
    }
  }
  if ((what & kState) && blockIdx.x == 0) {
    __syncthreads();  // one workgroup may write over what it has read
    for (int b = tid; b < p.B; b += 256) {
      const Row r = row_of(b);
      p.held_out[b] = served(r, b) ? r.have - r.back + r.take : r.have;
    }
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
};

// y = x / sqrt(mean(x^2) + eps) * w, its pairs turned by pos * turns[i] (a turn
// is 2 pi) and stretched by factor; everything in fp32, rounded once.
// One wave takes NH heads of one token (q heads, then k, then v): the angles
// depend on the token and the lane only and serve all of them.  The angle is
// exact at any position: pos * turns in 64-bit integers drops whole turns by
// itself, where pos * frequency in fp32 is off by 0.06 rad at a million; its top
// 32 bits go to the hardware's sine and cosine, which take turns.
template <int D, int NH, bool IL>
__global__ __launch_bounds__(256) void attn_rope_kernel(const RopeParams p) {
  constexpr int EPL = D / 64;  // elements per lane
  typedef typename RowVec<EPL>::type vec;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = p.Hq + 2 * p.Hkv;
  const uint32_t per_tok = (heads + NH - 1) / NH;
  const uint32_t item = blockIdx.x * 4u + wave;
  const uint32_t bt = item / per_tok;
  if (bt >= static_cast<uint32_t>(p.B) * p.T) return;  // wave-uniform
  const int h0 = static_cast<int>(item - bt * per_tok) * NH;
  const int b = static_cast<int>(bt / p.T), t = static_cast<int>(bt - static_cast<uint32_t>(b) * p.T);
  const int d0 = EPL * lane;

  vec raw[NH];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    const int h = min(h0 + n, heads - 1);
    const uint16_t* src;
    if (h < p.Hq) src = p.qg + bt * p.qg_ld + h * p.q_head;
    else if (h < p.Hq + p.Hkv) src = p.kn + bt * p.kv_ld + (h - p.Hq) * D;
    else src = p.vn + bt * p.kv_ld + (h - p.Hq - p.Hkv) * D;
    raw[n] = *reinterpret_cast<const vec*>(src + d0);
  }
  const bool norm = p.qw != nullptr;
  uint32_t qwr[EPL] = {}, kwr[EPL] = {};
  if (norm) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      if (p.wdt == GDN_DTYPE_F32) {
        qwr[e] = static_cast<const uint32_t*>(p.qw)[d0 + e];
        kwr[e] = static_cast<const uint32_t*>(p.kw)[d0 + e];
      } else {
        qwr[e] = static_cast<const uint16_t*>(p.qw)[d0 + e];
        kwr[e] = static_cast<const uint16_t*>(p.kw)[d0 + e];
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

  // sine and cosine of the lane's elements; the first of a pair takes -sine
  const int half = p.rot / 2;
  const bool lower = d0 < half;
  const int partner = lower ? lane + half / EPL : lane - half / EPL;
  float sn[EPL], cs[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    sn[e] = 0.0f;
    cs[e] = 1.0f;
    if (d0 + e < p.rot) {
      const int i = IL ? (d0 + e) / 2 : lower ? d0 + e : d0 + e - half;
      const uint64_t f = p.turns[i];
      const uint32_t phase = static_cast<uint32_t>(f >> 32) * pos + __umulhi(static_cast<uint32_t>(f), pos);
      const float x = static_cast<float>(static_cast<int32_t>(phase)) * 0x1p-32f;
      const float s = __builtin_amdgcn_sinf(x) * p.factor;
      sn[e] = (IL ? e % 2 == 0 : lower) ? -s : s;
      cs[e] = __builtin_amdgcn_cosf(x) * p.factor;
    }
  }
  auto weight = [&](uint32_t u) {
    return p.wdt == GDN_DTYPE_F32 ? __uint_as_float(u)
                                  : (p.wdt == GDN_DTYPE_BF16 ? bf16_to_f32(static_cast<uint16_t>(u))
                                                             : f16_to_f32(static_cast<uint16_t>(u)));
  };
  float qw[EPL], kw[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    qw[e] = norm ? weight(qwr[e]) : 1.0f;
    kw[e] = norm ? weight(kwr[e]) : 1.0f;
  }

  float r[NH];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const float x = bf16_to_f32(raw[n][e]);
      ss += x * x;
    }
    r[n] = norm ? rsqrtf(wave_sum(ss) / D + p.eps) : 1.0f;
  }
  vec out[NH];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    float x[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) x[e] = bf16_to_f32(raw[n][e]) * r[n] * (h0 + n < p.Hq ? qw[e] : kw[e]);
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const float other = IL ? x[e ^ 1] : __shfl(x[e], partner, 64);
      out[n][e] = f32_to_bf16(d0 + e < p.rot ? x[e] * cs[e] + other * sn[e] : x[e]);
    }
  }
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    const int h = h0 + n;
    if (h >= heads) return;  // wave-uniform
    if (h < p.Hq) {
      *reinterpret_cast<vec*>(p.q + (static_cast<int64_t>(bt) * p.Hq + h) * D + d0) = pad ? vec{} : out[n];
    } else if (!pad) {
      const bool is_k = h < p.Hq + p.Hkv;  // v goes into its slot as is
      const int hkv = h - p.Hq - (is_k ? 0 : p.Hkv);
      *reinterpret_cast<vec*>((is_k ? p.keys : p.values) + ((static_cast<int64_t>(page) * p.Hkv + hkv) * p.block + at) * D + d0) =
          is_k ? out[n] : raw[n];
    }
  }
}

// ------------------------------------------------------------ attention

// One launch covers a step: the workgroups of the shared prefix first (all rows
// of the batch, read once per row tile), then each row's own keys.
struct StepParams : PagedParams {
  int n_prefix, n_own;        // key ranges
  int len_prefix, len_own;    // keys of a range
  int prefix_tiles, own_tiles;  // row tiles; 0: the rows fit the 16 of attn_rows
};

// Up to 16 rows of kv-head hkv (of batch entry b, or of the whole batch) over key
// range `split`, by W waves.  Every wave takes 16 KT keys of a step of 16 KT W and
// keeps a softmax state of its own; nothing in the loop waits for another wave.
// K and V go to the wave's own 16 KB of LDS by direct loads of whole rows (K as
// fragments from memory, 64 bytes of a row at a time, took 1.6 times as long from
// a warm cache), their 16-byte granules swizzled on the way: K's by (key & 7), so
// that 16-byte fragment reads of 8 keys hit distinct banks, V's by 2 (key & 7), so
// that its transposed reads of 4 x 4 keys do.  K of the next step is asked for as
// soon as this one's scores are formed, V as soon as its products are: a CU has up
// to 128 KB in flight.  Bound by memory: a full cache of 64 rows of 4096 keys at 4
// kv-heads of 256 (1.07 GB) takes 164 us, 6.6 TB/s (without the hint that the keys
// are read once 186).
// Tiles of 32 rows in the same way (O and Q in 192 registers) were within 10% of
// attn_tile either way at 17 to 32 rows and slower beyond.
template <int D, int W>
constexpr int rows_lds() {
  constexpr int kv = W * 2 * 256 * 16 * 2, merge = W * 16 * D * 4 + 2 * W * 16 * 4;
  return kv > merge ? kv : merge;
}
template <int D, int W>
__device__ __forceinline__ void attn_rows(const PagedParams& p, unsigned char* smem, int b, int hkv, int split) {
  constexpr int KT = 256 / D;         // 16-key tiles per wave and step
  constexpr int KW = 16 * KT;         // keys per wave and step
  constexpr int KS = KW * W;          // keys per step
  constexpr int NS = D / 32, NJ = D / 16;
  constexpr int KROW = D / 8;         // 16-byte granules per row
  constexpr int LD = KW * KROW / 64;  // direct loads of 1 KB per wave, step and operand
  constexpr int STAGE = KW * D * 2;   // bytes
  const int g = p.Hq / p.Hkv;
  const int n_rows = tile_rows(p, g);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lq = lane >> 4;
  const int tokens = row_tokens(p, b);
  const int p0 = row_start(p, b, tokens);
  const KeyRange range = key_range(p, split, p0, tokens - 1, tokens > 0);
  const int k_lo = range.lo + KW * wave, k_hi = range.hi;  // this wave's keys: KW from k_lo, k_lo + KS, ..
  const int k_free = prefix_of(p) ? k_hi : min(p0 + 1, k_hi);  // keys below this are visible to every row
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
  const int row0 = lane / KROW, gran = lane % KROW;
  static_assert(64 % KROW == 0, "whole rows per load");
  constexpr int RL = 64 / KROW;  // rows per load
  // a row's own keys are read by one workgroup
  const bool once = !prefix_of(p) && !p.reread;
  auto load = [&](const uint16_t* pool, int i, uint32_t lds, int twist) {
    const int kb = k_lo + KS * i;
    const int64_t off = key_off<D>(p, b, hkv, kb, __builtin_amdgcn_readlane(pages, i - page0)) * 2;
    const u32x4 rsrc = buf_words(reinterpret_cast<const unsigned char*>(pool) + off, min(k_hi - kb, KW) * (D * 2));
#pragma unroll
    for (int c = 0; c < LD; ++c) {
      const int row = c * RL + row0;
      const uint32_t off = row * (D * 2) + (gran ^ (twist * (row & 7))) * 16;
      if (once) lds_dma16_once(rsrc, off, lds + c * 1024);
      else lds_dma16(rsrc, off, lds + c * 1024);
    }
  };

  if (n_step > 0) {
    load_pages(0);
    load(p.kc, 0, lds0, 1);
  }
  // lane lr's row: Q as the B operand of S^T = K Q^T
  const RowAt at = row_at(p, b, hkv, g, lr < n_rows ? lr : 0);
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
        a = mfma16(*reinterpret_cast<const bf16x8*>(ks + (16 * kt + lr) * (D * 2) + ((4 * s + lq) ^ (lr & 7)) * 16), qf[s], a);
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
  float* Os = reinterpret_cast<float*>(smem);  // [W][16][D]
  float* Ms = Os + W * 16 * D;                 // [W][16]
  float* Ls = Ms + W * 16;
#pragma unroll
  for (int j = 0; j < NJ; ++j) *reinterpret_cast<f32x4*>(&Os[(wave * 16 + lr) * D + 16 * j + 4 * lq]) = o[j];
  if (lq == 0) {
    Ms[wave * 16 + lr] = m;
    Ls[wave * 16 + lr] = l;
  }
  __syncthreads();
  constexpr int CW = D / (4 * W);  // columns per thread, in pieces of 4, 16 W apart
  static_assert(CW % 4 == 0, "whole pieces");
  const int mr = threadIdx.x / (4 * W), c0 = (threadIdx.x % (4 * W)) * 4;
  if (mr >= n_rows) return;
  const RowAt mat = row_at(p, b, hkv, g, mr);
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
      acc[c] += mw[w] * *reinterpret_cast<const f32x4*>(&Os[(w * 16 + mr) * D + c0 + 16 * W * c]);
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
  const int n_prefix = p.Hkv * p.n_prefix * max(p.prefix_tiles, 1);
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
  if (tiles == 0) attn_rows<D, W>(r, smem, b, hkv, split);
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

int lg2(int64_t x) {  // of a power of two, else -1
  return x > 0 && (x & (x - 1)) == 0 ? __builtin_ctzll(static_cast<uint64_t>(x)) : -1;
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
  if (B * T > INT32_MAX || n_blocks * block > INT32_MAX)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_paged_tables: tokens and slots must each be below 2^31");
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
  const int64_t groups = (B * T + 1023) / 1024;
  const unsigned grid = static_cast<unsigned>(groups < 1 ? 1 : groups > 512 ? 512 : groups);
  const bool in_place = held_out == held || n_free_out == n_free;
  hipLaunchKernelGGL(tables_kernel, dim3(grid), dim3(256), 0, st, p, grid > 1 && in_place ? kCells : kCells | kState);
  int rc = gdn_host::check_launch("gdn_paged_tables");
  if (rc != GDN_OK || !(grid > 1 && in_place)) return rc;
  hipLaunchKernelGGL(tables_kernel, dim3(1), dim3(256), 0, st, p, kState);
  return gdn_host::check_launch("gdn_paged_tables/state");
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
  if (rot < 0 || rot > D || rot % 2 != 0 || (!interleaved && rot % (2 * (D / 64)) != 0))
    return fail(GDN_ERR_UNSUPPORTED, "gdn_attn_rope: rotary dims %lld not supported for head dim %lld", (long long)rot,
                (long long)D);
  if ((q_norm_w == nullptr) != (k_norm_w == nullptr) || (q_norm_w && !gdn_host::dtype_ok(w_dtype)) || !(eps >= 0.0f))
    return fail(GDN_ERR_INVALID, "gdn_attn_rope: bad norm weights or eps");
  if (B * T == 0) return GDN_OK;
  if (!qg || !k_new || !v_new || !pos0 || (rot > 0 && !turns) || !q_out || !keys || !values)
    return fail(GDN_ERR_INVALID, "gdn_attn_rope: null pointer");
  if (B * T * (Hq + 2 * Hkv) > INT32_MAX || q_head > INT32_MAX)
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
  auto launch = [&](auto nh, auto il) {
    constexpr int NH = decltype(nh)::value;
    constexpr bool IL = decltype(il)::value;
    const dim3 grid(static_cast<unsigned>((B * T * ((Hq + 2 * Hkv + NH - 1) / NH) + 3) / 4));
    if (D == 256) hipLaunchKernelGGL((attn_rope_kernel<256, NH, IL>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((attn_rope_kernel<128, NH, IL>), grid, dim3(256), 0, st, p);
  };
  auto heads_per_wave = [&](auto il) {
    const int64_t rows = B * T * (Hq + 2 * Hkv);
    if (rows <= 4096) launch(std::integral_constant<int, 1>{}, il);
    else if (rows <= 16384) launch(std::integral_constant<int, 3>{}, il);
    else launch(std::integral_constant<int, 6>{}, il);
  };
  if (interleaved) heads_per_wave(std::true_type{});
  else heads_per_wave(std::false_type{});
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
                              int64_t n_own, void* workspace, size_t workspace_bytes, void* stream) {
  using gdn_host::fail;
  if (D != 128 && D != 256) return fail(GDN_ERR_UNSUPPORTED, "gdn_paged_attn: head dim must be 128 or 256 (got %lld)", (long long)D);
  const int lg = lg2(block);
  if (lg < 6 || lg > 20)
    return fail(GDN_ERR_UNSUPPORTED, "gdn_paged_attn: blocks must be powers of two from 64 to 2^20 keys (got %lld)", (long long)block);
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || n_blocks <= 0 || n_blocks > INT32_MAX ||
      table_ld <= 0 || table_ld > INT32_MAX || table_ld * block > INT32_MAX || T > table_ld * block ||
      kv_len_max > table_ld * block || shared < 0 || shared > table_ld ||
      kv_len_max < shared * block + (n_new ? 0 : T) || n_prefix < 0 || n_prefix > 65535 || n_own < 1 ||
      n_own > 65535 || (n_prefix > 0 && shared == 0))
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
  if (B > 65535 || B * T * Hq > INT32_MAX / 2 || Hkv * n_split > INT32_MAX ||
      B * Hkv * rows * n_split * (D + 2) > (int64_t(1) << 40))
    return fail(GDN_ERR_UNSUPPORTED, "gdn_paged_attn: problem too large");
  const size_t need = gdn_paged_attn_workspace_bytes(B, T, Hq, Hkv, D, n_split);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !gdn_host::aligned(workspace, 16)))
    return fail(GDN_ERR_INVALID, "gdn_paged_attn: workspace of %zu bytes is below the %zu needed for %lld key ranges",
                workspace_bytes, need, (long long)n_split);
  StepParams p;
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
  p.reread = n_prefix == 0 && shared > 0;
  auto range_len = [](int64_t keys, int64_t n) { return static_cast<int>(((keys + n - 1) / n + KB - 1) / KB * KB); };
  p.n_prefix = static_cast<int>(n_prefix);
  p.n_own = static_cast<int>(n_own);
  p.len_prefix = n_prefix > 0 ? range_len(p.key0, n_prefix) : 0;
  p.len_own = range_len(kv_len_max - p.key0, n_own);
  auto tiles_of = [](int64_t n) { return static_cast<int>(n <= 16 ? 0 : (n + PR - 1) / PR); };
  p.prefix_tiles = n_prefix > 0 ? tiles_of(B * rows) : 0;
  p.own_tiles = tiles_of(rows);
  const int64_t groups = Hkv * (n_prefix * (p.prefix_tiles > 1 ? p.prefix_tiles : 1) +
                                B * n_own * (p.own_tiles > 1 ? p.own_tiles : 1));
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
