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
  if (B > 65535 || Hkv > 65535 || (B * rows + PR - 1) / PR > 65535 || Hkv * n_split > INT32_MAX ||
      B * Hkv * rows * n_split * (D + 2) > (int64_t(1) << 40))
    return fail(GDN_ERR_UNSUPPORTED, "gdn_paged_attn: problem too large");
  const size_t need = gdn_paged_attn_workspace_bytes(B, T, Hq, Hkv, D, n_split);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !gdn_host::aligned(workspace, 16)))
    return fail(GDN_ERR_INVALID, "gdn_paged_attn: workspace of %zu bytes is below the %zu needed for %lld key ranges",
                workspace_bytes, need, (long long)n_split);
  PagedParams p;
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
  auto launch = [&](int64_t tile_rows, int64_t batch, int64_t keys_lo, int64_t keys_hi, int64_t n, int64_t split0) {
    p.key0 = static_cast<int>(n_prefix > 0 ? shared * block : 0);
    p.prefix = n_prefix > 0 && split0 == 0;
    p.split0 = static_cast<int>(split0);
    p.split_len = static_cast<int>(((keys_hi - keys_lo + n - 1) / n + KB - 1) / KB * KB);
    if (tile_rows <= 16) {
      const dim3 grid(static_cast<unsigned>(n), static_cast<unsigned>(Hkv), static_cast<unsigned>(batch));
      if (D == 256) hipLaunchKernelGGL((attn_fwd_kernel<256, 1, PagedParams>), grid, dim3(256), 0, st, p);
      else hipLaunchKernelGGL((attn_fwd_kernel<128, 1, PagedParams>), grid, dim3(256), 0, st, p);
    } else {
      const int64_t tiles = (tile_rows + PR - 1) / PR;
      const dim3 grid(static_cast<unsigned>(Hkv * n), static_cast<unsigned>(tiles), static_cast<unsigned>(batch));
      if (D == 256) hipLaunchKernelGGL((attn_prefill_kernel<256, 2, PagedParams>), grid, dim3(512), 0, st, p);
      else hipLaunchKernelGGL((attn_prefill_kernel<128, 1, PagedParams>), grid, dim3(256), 0, st, p);
    }
    return gdn_host::check_launch("gdn_paged_attn");
  };
  const int64_t key0 = n_prefix > 0 ? shared * block : 0;
  if (n_prefix > 0) {
    const int rc = launch(B * rows, 1, 0, key0, n_prefix, 0);
    if (rc != GDN_OK) return rc;
  }
  const int rc = launch(rows, B, key0, kv_len_max, n_own, n_prefix);
  if (rc != GDN_OK || n_split == 1) return rc;
  const dim3 cgrid(static_cast<unsigned>((B * Hkv * rows + 3) / 4));
  if (D == 256) hipLaunchKernelGGL((attn_combine_kernel<256, PagedParams>), cgrid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((attn_combine_kernel<128, PagedParams>), cgrid, dim3(256), 0, st, p);
  return gdn_host::check_launch("gdn_paged_attn/combine");
}
