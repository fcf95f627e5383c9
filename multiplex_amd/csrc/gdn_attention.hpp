// Attention kernels over cached keys and values on gfx950 (bf16 MFMA, online
// softmax in fp32), shared by the dense cache (gdn_attention.hip) and the paged
// one (gdn_paged.hip): the parameter block P says where a row's keys lie.
#pragma once

#include <cfloat>
#include <climits>

#include "gdn_common.hpp"

namespace {

using namespace gdn;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int KB = 64;  // keys per staged block

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma16k16(i16x4 a, i16x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x * kLog2e));
}

// A row's first position, clamped so that its T new tokens fit in the cache
// (offsets come from device memory and are not validated on the host).
__device__ __forceinline__ int first_pos(const int32_t* pos0, int b, int T, int cap) {
  return min(max(pos0[b], 0), cap - T);
}

// EPL bf16 elements of a row at any 2-byte address, as one load / store (callers
// may pass rows at any element offset; the hardware takes unaligned dwords).
template <int EPL>
struct RowVec {
  typedef uint16_t type __attribute__((ext_vector_type(EPL), aligned(2)));
};

// ------------------------------------------------------------ attn_fwd

struct AttnParams {
  static constexpr bool kPaged = false;
  const uint16_t* q;   // [B, T, Hq, D]
  const uint16_t* qg;  // gate source [B, T, Hq, 2D] (gate = second half of a head; token stride qg_ld) or null
  int64_t qg_ld;
  const uint16_t* kc;  // [B, Hkv, cap, D]
  const uint16_t* vc;
  const int32_t* pos0;  // [B]
  uint16_t* out;        // [B, T, Hq, D]
  float* part;          // split partials: O [B, Hkv, rows_pad, n_split, D], then m and l [.., n_split]
  int B, T, Hq, Hkv, cap;
  int n_split, split_len, rows_pad;
  float scale_log2;  // softmax scale * log2(e)
};

// The paged cache: pools of blocks [n_blocks, Hkv, 2^lg, D] in kc and vc, a
// table of a row's blocks, and up to T new tokens a row.  A launch covers either
// each row's own keys from position key0 on, or (prefix) the keys below key0,
// which every row's table lists alike: then a kv-head's tile rows are the whole
// batch's, [B, T, group], none of them is masked, and the keys are read once for
// all.  A block holds whole steps of KB keys, and key0 is a block's start.
struct PagedParams : AttnParams {
  static constexpr bool kPaged = true;
  const int32_t* table;  // [B, table_ld]
  const int32_t* n_new;  // [B] or null: T
  int table_ld, lg, n_blocks, key0, prefix;
  int split0;  // the launch's first key range of the row's n_split
  int pos_min;  // the shared keys, which every row has; above key0, rows read them too as their own
  int new_max;  // T, or the keys that a table lists behind the shared ones, where they are fewer (n_new is read as no more)
};

// A value that no kernel of this library's call writes, by a scalar load where
// its address is the wave's (also behind inline assembly that may write memory).
__device__ __forceinline__ int32_t const_i32(const int32_t* p, int64_t i) {
  return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p))[i];
}

// The new tokens of a row.
template <class P>
__device__ __forceinline__ int row_tokens(const P& p, int b) {
  if constexpr (P::kPaged) return p.n_new != nullptr ? min(max(const_i32(p.n_new, b), 0), p.new_max) : p.T;
  else return p.T;
}

// Position of a row's first new token: the keys it finds in the cache, clamped
// like first_pos (and not below the keys all rows share, however they are read).
template <class P>
__device__ __forceinline__ int row_start(const P& p, int b, int tokens) {
  if constexpr (P::kPaged) return p.prefix ? p.key0 : min(max(const_i32(p.pos0, b), p.pos_min), p.cap - tokens);
  else return first_pos(p.pos0, b, p.T, p.cap);
}

// Tile rows of a kv-head in one launch's batch entry, and where tile row r lies:
// batch row b, token t, query head hq, and the row's index among b's.
template <class P>
__device__ __forceinline__ bool prefix_of(const P& p) {
  if constexpr (P::kPaged) return p.prefix != 0;
  else return false;
}
template <class P>
__device__ __forceinline__ int tile_rows(const P& p, int g) {
  return prefix_of(p) ? p.B * p.T * g : p.T * g;
}
struct RowAt {
  int b, t, hq, row;
};
template <class P>
__device__ __forceinline__ RowAt row_at(const P& p, int b, int hkv, int g, int r) {
  if constexpr (P::kPaged) {
    if (p.prefix) {
      b = r / (p.T * g);
      r -= b * (p.T * g);
    }
  }
  return {b, r / g, hkv * g + r % g, r};
}

// The keys [lo, hi) of a launch's key range, for tile rows whose last new token is
// t_last (any: there is one).
struct KeyRange {
  int lo, hi;
};
template <class P>
__device__ __forceinline__ KeyRange key_range(const P& p, int split, int p0, int t_last, bool any) {
  if constexpr (P::kPaged) {
    const int lo = (p.prefix ? 0 : p.key0) + split * p.split_len;
    return {lo, p.prefix ? min(p.key0, lo + p.split_len) : any ? min(p0 + t_last + 1, lo + p.split_len) : lo};
  } else {
    const int lo = split * p.split_len;
    return {lo, min(p0 + t_last + 1, lo + p.split_len)};
  }
}

// Element offset of key kb's row (the first of a step of KB keys) in a pool or
// cache.  A table entry outside the pool reads another block, never past it.
template <class P>
__device__ __forceinline__ int block_of(const P& p, int b, int kb) {
  if constexpr (P::kPaged) {
    const int page = const_i32(p.table, static_cast<int64_t>(p.prefix ? 0 : b) * p.table_ld + min(kb >> p.lg, p.table_ld - 1));
    return min(max(page, 0), p.n_blocks - 1);
  } else {
    return 0;
  }
}
template <int D, class P>
__device__ __forceinline__ int64_t key_off(const P& p, int b, int hkv, int kb, int page) {
  if constexpr (P::kPaged)
    return (((static_cast<int64_t>(page) * p.Hkv + hkv) << p.lg) + (kb & ((1 << p.lg) - 1))) * D;
  else
    return ((static_cast<int64_t>(b) * p.Hkv + hkv) * p.cap + kb) * D;
}

// Index of the launch's range among the row's n_split ranges.
template <class P>
__device__ __forceinline__ int split_at(const P& p, int split) {
  if constexpr (P::kPaged) return p.split0 + split;
  else return split;
}

// Partial-state addressing for split keys.
__device__ __forceinline__ int64_t part_row(const AttnParams& p, int b, int hkv, int r) {
  return ((static_cast<int64_t>(b) * p.Hkv + hkv) * p.rows_pad + r) * p.n_split;
}

// Final value of one output element pair / quad: o / l, times the gate.
template <int D>
__device__ __forceinline__ void store_out4(const AttnParams& p, int b, int t, int hq, int d, f32x4 o, float inv_l) {
  const int64_t bt = static_cast<int64_t>(b) * p.T + t;
  const int64_t row = bt * p.Hq + hq;
  f32x4 y = o * inv_l;
  if (p.qg != nullptr) {
    const u32x2 gg = *reinterpret_cast<const u32x2*>(p.qg + bt * p.qg_ld + hq * 2 * D + D + d);
    y[0] *= sigmoid(__uint_as_float(gg.x << 16));
    y[1] *= sigmoid(__uint_as_float(gg.x & 0xffff0000u));
    y[2] *= sigmoid(__uint_as_float(gg.y << 16));
    y[3] *= sigmoid(__uint_as_float(gg.y & 0xffff0000u));
  }
  *reinterpret_cast<u32x2*>(p.out + row * D + d) = u32x2{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3])};
}

// A lane's N pieces of 4 of one output row, STEP columns apart: o / l times the gate, whose loads are all
// issued before the first is used.  (l = 0: every score is -inf, whose softmax is NaN.)
// `row` is the row of out: token times Hq plus head.
template <int D, int N, int STEP>
__device__ __forceinline__ void store_row(const AttnParams& p, int row, int d, const f32x4* o, float l) {
  uint16_t* out = p.out + static_cast<int64_t>(row) * D + d;
  const float inv_l = 1.0f / l;
  if (p.qg == nullptr) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const f32x4 y = o[n] * inv_l;
      *reinterpret_cast<u32x2*>(out + STEP * n) = u32x2{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3])};
    }
    return;
  }
  const int bt = row / p.Hq, hq = row - bt * p.Hq;
  const uint16_t* qg = p.qg + bt * p.qg_ld + hq * 2 * D + D + d;
  u32x2 gate[N];
#pragma unroll
  for (int n = 0; n < N; ++n) gate[n] = *reinterpret_cast<const u32x2*>(qg + STEP * n);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    f32x4 y = o[n] * inv_l;
    y[0] *= sigmoid(__uint_as_float(gate[n].x << 16));
    y[1] *= sigmoid(__uint_as_float(gate[n].x & 0xffff0000u));
    y[2] *= sigmoid(__uint_as_float(gate[n].y << 16));
    y[3] *= sigmoid(__uint_as_float(gate[n].y & 0xffff0000u));
    *reinterpret_cast<u32x2*>(out + STEP * n) = u32x2{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3])};
  }
}

// A padded token's output.
template <int D>
__device__ __forceinline__ void store_zero4(const AttnParams& p, int b, int t, int hq, int d) {
  *reinterpret_cast<u32x2*>(p.out + ((static_cast<int64_t>(b) * p.T + t) * p.Hq + hq) * D + d) = u32x2{0u, 0u};
}

template <int D, int RT>
__global__ __launch_bounds__(256) void attn_fwd_kernel(const AttnParams p) {
  constexpr int KP = D + 8;   // K row stride (bf16): 16-byte fragment reads of 16 rows hit distinct banks
  constexpr int VP = D + 16;  // V row stride: the transposed reads of 4 rows hit distinct banks
  constexpr int KT = RT == 4 ? 4 : 1;  // 16-key tiles per wave and block
  constexpr int NS = D / 32;           // k-steps of q . k
  constexpr int NJ = D / 16;           // 16-wide d tiles of the output
  constexpr int CPT = KB * D / 8 / 256;  // 16-byte chunks per thread of a K (or V) block

  const int b = blockIdx.z;
  const int hkv = blockIdx.y % p.Hkv, rb = blockIdx.y / p.Hkv;
  const int split = blockIdx.x;
  const int g = p.Hq / p.Hkv;
  const int n_rows = p.T * g;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lq = lane >> 4;
  const int p0 = first_pos(p.pos0, b, p.T, p.cap);

  const int row0 = rb * 16 * RT;
  const int t_last = min((row0 + 16 * RT - 1) / g, p.T - 1);
  const int k_lo = split * p.split_len;
  const int k_hi = min(p0 + t_last + 1, k_lo + p.split_len);  // keys of this workgroup: [k_lo, k_hi)
  const int rt = RT == 4 ? wave : 0;
  const int sub = RT == 4 ? 0 : wave;  // first 16-key tile of this wave in each block

  // this wave's 16 rows (lane lr's row): Q as the B operand of S^T = K Q^T
  const int r = row0 + 16 * rt + lr;
  const bool row_ok = r < n_rows;
  const int t = row_ok ? r / g : 0;
  const int hq = hkv * g + (row_ok ? r % g : 0);
  const int kmax = p0 + t;  // last key row r may see
  bf16x8 qf[NS];
  {
    const uint16_t* qrow = p.q + ((static_cast<int64_t>(b) * p.T + t) * p.Hq + hq) * D;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(qrow + 32 * s + 8 * lq);
      qf[s] = __builtin_bit_cast(bf16x8, row_ok ? v : u32x4{0u, 0u, 0u, 0u});
    }
  }

  __shared__ __align__(16) unsigned char smem[KB * (KP + VP) * 2];
  uint16_t(*Ks)[KP] = reinterpret_cast<uint16_t(*)[KP]>(smem);
  uint16_t(*Vs)[VP] = reinterpret_cast<uint16_t(*)[VP]>(smem + KB * KP * 2);

  // the next block, in flight: chunk c = tid + 256 i is row c / (D/8), columns (c % (D/8)) * 8 ..
  // The cache is read with nontemporal loads: each step streams it once, and at
  // decode sizes (1 GB at B=64 and 4096 positions) it cannot stay in the
  // last-level cache, whose allocation on every read cost 15% (180.4 against
  // 152.8 us at B=64).
  u32x4 kr[CPT], vr[CPT];
  const int64_t head_base = (static_cast<int64_t>(b) * p.Hkv + hkv) * p.cap * D;
  auto load_blk = [&](int kb) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = tid + 256 * i;
      const int row = c / (D / 8), col = (c % (D / 8)) * 8;
      const int key = kb + row;
      const int64_t off = head_base + static_cast<int64_t>(min(key, k_hi - 1)) * D + col;  // in bounds: k_hi <= cap
      kr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p.kc + off));
      vr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p.vc + off));
    }
  };
  auto store_blk = [&](int kb) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = tid + 256 * i;
      const int row = c / (D / 8), col = (c % (D / 8)) * 8;
      const bool ok = kb + row < k_hi;  // keys past the range read as zero (the cache there is unset)
      const u32x4 z = {0u, 0u, 0u, 0u};
      *reinterpret_cast<u32x4*>(&Ks[row][col]) = ok ? kr[i] : z;
      *reinterpret_cast<u32x4*>(&Vs[row][col]) = ok ? vr[i] : z;
    }
  };

  float m = -INFINITY, l = 0.0f;  // running max (log2 units) and this lane's share of the sum
  f32x4 o[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int nblk = k_hi > k_lo ? (k_hi - k_lo + KB - 1) / KB : 0;
  if (nblk > 0) load_blk(k_lo);
  for (int blk = 0; blk < nblk; ++blk) {
    const int kb = k_lo + KB * blk;
    __syncthreads();  // the previous block's reads are done
    store_blk(kb);
    __syncthreads();
    if (blk + 1 < nblk) load_blk(kb + KB);

    // S^T = K Q^T for this wave's key tiles: lane (r, q) holds keys 16 kt + 4q + i of row r
    f32x4 sc[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < NS; ++s)
        a = mfma16(*reinterpret_cast<const bf16x8*>(&Ks[16 * (sub + kt) + lr][32 * s + 8 * lq]), qf[s], a);
      sc[kt] = a;
    }
    float mb = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = kb + 16 * (sub + kt) + 4 * lq + i;
        const bool ok = row_ok && key <= kmax && key < k_hi;
        sc[kt][i] = ok ? sc[kt][i] * p.scale_log2 : -INFINITY;
        mb = fmaxf(mb, sc[kt][i]);
      }
    mb = fmaxf(mb, __shfl_xor(mb, 16, 64));
    mb = fmaxf(mb, __shfl_xor(mb, 32, 64));
    const float m_new = fmaxf(m, mb);
    const float m_use = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - m_use);
    m = m_new;
    float ps = 0.0f;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[kt][i] = __builtin_amdgcn_exp2f(sc[kt][i] - m_use);
        ps += sc[kt][i];
      }
    l = l * alpha + ps;
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] *= alpha;

    // O^T += V^T P^T (P as bf16; V^T by transposed LDS reads)
    if constexpr (RT == 4) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        // k-slots: keys 32 ks + 4q + (0..3), then 32 ks + 16 + 4q + (0..3) -- the rows of
        // accumulator tiles 2 ks and 2 ks + 1 held by lane group q
        const bf16x8 pb = __builtin_bit_cast(
            bf16x8, u32x4{pk_bf16(sc[2 * ks][0], sc[2 * ks][1]), pk_bf16(sc[2 * ks][2], sc[2 * ks][3]),
                          pk_bf16(sc[2 * ks + 1][0], sc[2 * ks + 1][1]), pk_bf16(sc[2 * ks + 1][2], sc[2 * ks + 1][3])});
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint16_t* va = &Vs[32 * ks + 4 * lq + (lr >> 2)][16 * j + 4 * (lr & 3)];
          const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(va));
          const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(va + 16 * VP));
          const bf16x8 vt = __builtin_bit_cast(bf16x8, i16x8(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)));
          o[j] = mfma16(vt, pb, o[j]);
        }
      }
    } else {
      const u32x2 pw = {pk_bf16(sc[0][0], sc[0][1]), pk_bf16(sc[0][2], sc[0][3])};
      const i16x4 pb = __builtin_bit_cast(i16x4, pw);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint16_t* va = &Vs[16 * sub + 4 * lq + (lr >> 2)][16 * j + 4 * (lr & 3)];
        o[j] = mfma16k16(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(va)), pb, o[j]);
      }
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  const bool split_out = p.n_split > 1;
  if constexpr (RT == 4) {
    // lane (r, q) holds O[row r][16 j + 4 q + i]
    if (!row_ok) return;
    if (split_out) {
      const int64_t pr = part_row(p, b, hkv, r) + split;
      float* po = p.part + pr * D;
#pragma unroll
      for (int j = 0; j < NJ; ++j) *reinterpret_cast<f32x4*>(po + 16 * j + 4 * lq) = o[j];
      if (lq == 0) {
        float* ml = p.part + static_cast<int64_t>(p.B) * p.Hkv * p.rows_pad * p.n_split * D;
        const int64_t n_part = static_cast<int64_t>(p.B) * p.Hkv * p.rows_pad * p.n_split;
        ml[pr] = m;
        ml[n_part + pr] = l;
      }
      return;
    }
    const float inv_l = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) store_out4<D>(p, b, t, hq, 16 * j + 4 * lq, o[j], inv_l);
  } else {
    // merge the four waves' states for the tile's 16 rows (the K/V buffers are free)
    __syncthreads();
    float* Os = reinterpret_cast<float*>(smem);  // [4][16][D]
    float* Ms = Os + 4 * 16 * D;                 // [4][16]
    float* Ls = Ms + 4 * 16;
    static_assert((4 * 16 * D + 2 * 64) * 4 <= KB * (KP + VP) * 2, "merge buffers must fit in the K/V blocks");
#pragma unroll
    for (int j = 0; j < NJ; ++j) *reinterpret_cast<f32x4*>(&Os[(wave * 16 + lr) * D + 16 * j + 4 * lq]) = o[j];
    if (lq == 0) {
      Ms[wave * 16 + lr] = m;
      Ls[wave * 16 + lr] = l;
    }
    __syncthreads();
    // thread: row tid / 16, columns (tid % 16) * D/16 ..
    constexpr int CW = D / 16;
    const int mr = tid >> 4, c0 = (tid & 15) * CW;
    const int rr = row0 + mr;
    if (rr >= n_rows) return;
    float mw[4], ms = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      mw[w] = Ms[w * 16 + mr];
      ms = fmaxf(ms, mw[w]);
    }
    const float m_use = ms == -INFINITY ? 0.0f : ms;
    float sw[4], lsum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      sw[w] = __builtin_amdgcn_exp2f(mw[w] - m_use);
      lsum += sw[w] * Ls[w * 16 + mr];
    }
    if (split_out) {
      const int64_t pr = part_row(p, b, hkv, rr) + split;
      float* po = p.part + pr * D;
#pragma unroll
      for (int c = 0; c < CW; c += 4) {
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) acc += sw[w] * *reinterpret_cast<const f32x4*>(&Os[(w * 16 + mr) * D + c0 + c]);
        *reinterpret_cast<f32x4*>(po + c0 + c) = acc;
      }
      if ((tid & 15) == 0) {
        float* ml = p.part + static_cast<int64_t>(p.B) * p.Hkv * p.rows_pad * p.n_split * D;
        const int64_t n_part = static_cast<int64_t>(p.B) * p.Hkv * p.rows_pad * p.n_split;
        ml[pr] = ms;
        ml[n_part + pr] = lsum;
      }
      return;
    }
    const float inv_l = lsum > 0.0f ? 1.0f / lsum : 0.0f;
    const int tt = rr / g, hh = hkv * g + rr % g;
#pragma unroll
    for (int c = 0; c < CW; c += 4) {
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < 4; ++w) acc += sw[w] * *reinterpret_cast<const f32x4*>(&Os[(w * 16 + mr) * D + c0 + c]);
      store_out4<D>(p, b, tt, hh, c0 + c, acc, inv_l);
    }
  }
}

// Causal prefills of at least kPrefillRows rows per kv-head: a workgroup owns
// 128 rows in four row groups of 32, so every K or V fragment a wave reads
// from LDS feeds two 16-row MFMA tiles.  64-key blocks are double-buffered in
// LDS and a block costs one barrier:
//   K  goes in by direct global -> LDS loads (each lane's 16 bytes land at
//      16 * lane past the wave's base), rows of D bf16 whose 16-byte granules
//      are XOR-swizzled by (key & 7), so the fragment reads of 8 consecutive
//      keys hit distinct banks;
//   V  is transposed in registers on its way in: Vt[d][position], with the
//      keys of each 32-key group in the k-slot order of the P^T operand
//      (position 8q + 4h + i holds key 16h + 4q + i), so that a V^T fragment
//      is one 16-byte read, like K's; rows of 64 positions whose 16-byte
//      granules are XOR-swizzled by (d & 7), which keeps both the fragment
//      reads and the 8-byte transposed writes free of bank conflicts.  (Transposed LDS reads of a [key][d]
//      block deliver about 45 bytes per clock per CU, against 128 for 16-byte
//      reads.)  Its loads are issued one block ahead of the transpose.
// KG = 2 (head dim 256, whose workgroup fills a CU's LDS): eight waves, two
// per SIMD, the two of a row group taking 32 keys of every block each with a
// softmax state of their own, merged in LDS at the end.  One wave's MFMAs
// then run beside the other's exponentials: a single wave issues a 16x16x32
// MFMA every 9.6 ns at best and two share a SIMD at 7.6 ns each, with two or
// three vector instructions per MFMA free.  Both must fit in 256 registers
// each without a spill (a reload per block waits for every load in flight:
// +9% per fragment), which is why two k-steps of q stay in LDS and few
// fragments are in flight.  KG = 1 (head dim 128): four waves, and two
// workgroups share a CU.
// Measured at 16 query and 4 kv-heads of 256: 4096 tokens 195 -> 165 us
// (840 TFLOP/s), 512 tokens over a 4096-token prefix in one key range 160 ->
// 128 us; four waves with the next block's scores computed between this
// block's exponentials, in registers enough for both, took 209 and 172 us.
// Few rows leave CUs idle, so the keys may be split over workgroups too
// (n_split; 512 tokens over 4096 in four ranges: 60 us with the combine).
// The softmax max is raised only when a row's block max exceeds it by more
// than 8 (log2 units; P stays below 2^8), which skips the rescale of the
// output on most blocks, and only blocks that cross the diagonal or the end
// of the keys are masked.  Workgroups with the longest key ranges go first.

// A raw buffer descriptor of `bytes` bytes at `base` (wave-uniform): reads past its end return zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buf_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(bytes), 0x00020000);
}

// Max / sum over the four 16-lane rows of a wave (lanes r, r + 16, r + 32, r + 48), by the
// gfx950 row-swap moves (VALU, no LDS round trip): permlane16_swap(x, x) yields the even and the
// odd rows, permlane32_swap(x, x) the low and the high halves, each in both places.
__device__ __forceinline__ float rows_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float rows_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Max over the 64 lanes.
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp_f<GDN_DPP_QUAD_XOR1>(x));
  x = fmaxf(x, dpp_f<GDN_DPP_QUAD_XOR2>(x));
  x = fmaxf(x, dpp_f<GDN_DPP_HALF_MIRROR>(x));
  x = fmaxf(x, dpp_f<GDN_DPP_ROW_MIRROR>(x));
  return rows_max(x);
}

constexpr int kPrefillRows = 512;  // rows (tokens x heads of a group) per kv-head from which it is used
constexpr int PR = 128;            // rows per workgroup
constexpr int VTP = KB;            // Vt row stride (bf16); 16-byte granules XOR-swizzled by (d & 7)
// bytes between 8 rows of K and the next 8.  A fragment's read takes 16 rows' granules a cycle: XOR-swizzled by
// (key & 7) they lie in half of the banks, the pad moves every other 8 rows to the other half (279 -> 480 B/ns a CU)
constexpr int K_PAD = 128;
template <int D>
constexpr int k_stage() { return KB * D * 2 + KB / 8 * K_PAD; }

// k-steps of q kept in LDS: as many as leave the loop without a spill.  They are spread over the 8 steps, so that one
// pair of registers takes each in while the products of the steps between are formed (as the last steps of all, waited
// for, 4 x 512 tokens behind 4096 keys took 131 us, not 129.6).
template <int KG, class P>
constexpr int q_lds_steps() { return KG == 2 ? (P::kPaged ? 3 : 2) : 0; }
// QL of 8 steps: 1, 4, 7 or 2, 6.  The slot of step s in LDS (-1: it is in registers), and the steps before s that
// are in registers.
constexpr int q_slot(int ql, int s) {
  const int step = ql == 3 ? 3 : 4, first = ql == 3 ? 1 : 2;
  return ql > 0 && s % step == first ? s / step : -1;
}
constexpr int q_reg(int ql, int s) {
  int n = 0;
  for (int i = 0; i < s; ++i) n += q_slot(ql, i) < 0;
  return n;
}
template <int D, int KG, class P>
constexpr int tile_lds() {
  return 2 * (k_stage<D>() + D * VTP * 2) + (KG == 2 ? 8 * 128 * 4 : 0) + 4 * 2 * q_lds_steps<KG, P>() * 1024 +
         (P::kPaged ? 3 * PR * 4 : 0);
}

// Tile rb of kv-head hkv's rows of batch entry b over key range `split`, by 256 * KG threads with
// tile_lds<D, KG, P>() bytes of LDS.
template <int D, int KG, class P>
__device__ __forceinline__ void attn_tile(const P& p, unsigned char* smem, int b, int hkv, int rb, int split) {
  constexpr int NT = 256 * KG;                // threads
  constexpr int NS = D / 32;                  // k-steps of q . k
  constexpr int NJ = D / 16;                  // 16-wide d tiles of the output
  constexpr int KTW = 4 / KG;                 // 16-key tiles of a block per wave
  constexpr int KSW = 2 / KG;                 // 32-key groups of a block per wave
  constexpr int KROW = D / 8;                 // 16-byte granules per K row
  constexpr int KDMA = KB * KROW / NT;        // direct loads per thread and K block
  constexpr int VPAIRS = (KB / 4) * KROW / NT;  // (key quad, d octet) pairs per thread and V block
  constexpr int KSTAGE = k_stage<D>();        // bytes
  constexpr int VSTAGE = D * VTP * 2;
  static_assert(KDMA * NT == KB * KROW && VPAIRS * NT == (KB / 4) * KROW, "block must split evenly over the threads");
  static_assert(KDMA <= NS && 4 * VPAIRS <= NS, "at most one K and one V load per k-step");

  constexpr int QL = q_lds_steps<KG, P>();
  constexpr int kMl = KG == 2 ? 8 * 128 * 4 : 0;  // the waves' (m, l) for the merge
  static_assert(tile_lds<D, KG, P>() == 2 * (KSTAGE + VSTAGE) + kMl + 4 * 2 * QL * 1024 + (P::kPaged ? 3 * PR * 4 : 0),
                "LDS layout");

  const int g = p.Hq / p.Hkv;
  const int n_rows = tile_rows(p, g);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = wave & 3, kh = wave >> 2;  // the wave's 32 rows of the workgroup's, and its keys of each block
  const int lr = lane & 15, lq = lane >> 4;
  const int tokens = row_tokens(p, b);
  const int p0 = row_start(p, b, tokens);

  const int row0 = rb * PR;
  const int t_last = min((row0 + PR - 1) / g, tokens - 1);
  const KeyRange keys = key_range(p, split, p0, t_last, row0 / g < tokens);
  const int k_lo = keys.lo, k_hi = keys.hi;  // keys of this workgroup: [k_lo, k_hi)
  const int k_free = prefix_of(p) ? k_hi : min(p0 + row0 / g + 1, k_hi);  // keys below this are visible to every row
  const int nblk = k_hi > k_lo ? (k_hi - k_lo + KB - 1) / KB : 0;

  // the wave's two 16-row tiles; rows past the end compute on q = 0 and are not stored.  QL k-steps of q are
  // kept in LDS (both waves of a row group read one copy)
  static_assert(QL == 0 || (NS == 8 && q_reg(QL, NS) == NS - QL), "steps of q in LDS");
  auto q_lds = [&](int rt, int slot) {
    return reinterpret_cast<bf16x8*>(smem + 2 * (KSTAGE + VSTAGE) + kMl) + ((rg * 2 + rt) * QL + slot) * 64 + lane;
  };
  int kmax[2];
  bf16x8 qf[2][NS - QL];
  // The paged form's rows, once per workgroup (several divisions each): their row of q and out (-1: none), the
  // last key they may see (-1: none, a padded token) and their row of the partial results.
  int* row_out = reinterpret_cast<int*>(smem + tile_lds<D, KG, P>()) - 3 * PR;
  int* row_kmax = row_out + PR;
  int* row_part = row_kmax + PR;
  auto find_rows = [&]() {
    if (tid < PR) {
      const int r = row0 + tid;
      const RowAt at = row_at(p, b, hkv, g, min(r, n_rows - 1));
      row_out[tid] = r < n_rows ? (at.b * p.T + at.t) * p.Hq + at.hq : -1;
      row_kmax[tid] = r < n_rows && (prefix_of(p) || at.t < tokens) ? (prefix_of(p) ? INT_MAX : p0 + at.t) : -1;
      row_part[tid] = (at.b * p.Hkv + hkv) * p.rows_pad + at.row;
    }
  };
  auto load_q = [&]() {
    if constexpr (P::kPaged) {
      // whole rows straight into the V stages' LDS, as K's blocks are, then as fragments from there (as fragments
      // from memory, 64 bytes of a row at a time, a workgroup takes 1.8 us more at D = 256; at 128 as long)
      static_assert(PR * D * 2 <= 2 * VSTAGE, "the rows must fit in the V stages");
      constexpr int RL = 64 / KROW, QI = PR / (NT / KROW);  // rows per load, loads per wave
      const int first = __builtin_amdgcn_readfirstlane(row_out[0]);
      const int last = __builtin_amdgcn_readfirstlane(row_out[min(PR, n_rows - row0) - 1]);
      const u32x4 rsrc = buf_words(p.q + static_cast<int64_t>(first) * D, (last - first + 1) * (D * 2));
      const uint32_t qs = __builtin_amdgcn_readfirstlane(
          static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem)) + 2 * KSTAGE + wave * (QI * 1024));
#pragma unroll
      for (int i = 0; i < QI; ++i) {
        const int r = (wave * QI + i) * RL + lane / KROW;
        const uint32_t row = max(row_out[r], first) - first;  // (past the end: the first, not stored)
        lds_dma16(rsrc, row * (D * 2) + (((lane % KROW) ^ (r & 15)) * 16), qs + i * 1024);
      }
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" : : : "memory");
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        const int r = 32 * rg + 16 * rt + lr;
        kmax[rt] = row_kmax[r];
        const bool ok = kmax[rt] >= 0;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(smem + 2 * KSTAGE + r * (D * 2) + ((4 * s + lq) ^ lr) * 16);
          const bf16x8 f = __builtin_bit_cast(bf16x8, ok ? x : u32x4{0u, 0u, 0u, 0u});
          if (q_slot(QL, s) < 0) qf[rt][q_reg(QL, s)] = f;
          else if (kh == 0) *q_lds(rt, q_slot(QL, s)) = f;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");  // the stages are free
      return;
    }
    u32x4 v[2][NS];
    bool ok[2];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      const int r = row0 + 32 * rg + 16 * rt + lr;
      const RowAt at = row_at(p, b, hkv, g, min(r, n_rows - 1));
      ok[rt] = r < n_rows;
      const int hq = ok[rt] ? at.hq : hkv * g;
      kmax[rt] = p0 + at.t;
      const uint16_t* qrow = p.q + ((static_cast<int64_t>(at.b) * p.T + at.t) * p.Hq + hq) * D;
#pragma unroll
      for (int s = 0; s < NS; ++s) v[rt][s] = *reinterpret_cast<const u32x4*>(qrow + 32 * s + 8 * lq);
    }
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const bf16x8 f = __builtin_bit_cast(bf16x8, ok[rt] ? v[rt][s] : u32x4{0u, 0u, 0u, 0u});
        if (q_slot(QL, s) < 0) qf[rt][q_reg(QL, s)] = f;
        else if (kh == 0) *q_lds(rt, q_slot(QL, s)) = f;
      }
  };
  if constexpr (!P::kPaged) load_q();

  // K and V blocks are read through descriptors that end at the range's last
  // key, so the lane offsets are constants and keys past the range (masked
  // below) read as zeros
  const int64_t head = P::kPaged ? 0 : (static_cast<int64_t>(b) * p.Hkv + hkv) * p.cap * D;
  const unsigned char* kc_head = reinterpret_cast<const unsigned char*>(p.kc + head);
  const unsigned char* vc_head = reinterpret_cast<const unsigned char*>(p.vc + head);
  // The paged cache's step i lies where the table says: lane l holds the block of step page0 + l, so that a
  // step's is one lane's read, and no load for it is among the loop's.
  int page0 = 0, pages = 0;
  auto load_pages = [&](int blk) {
    page0 = blk;
    const int kb = min(k_lo + KB * (blk + lane), k_hi - 1);
    pages = nblk > 0 ? block_of(p, b, kb) : 0;
  };
  // byte offset of the step of keys at kb (a whole number of steps past k_lo)
  auto step_off = [&](int kb) -> int64_t {
    if constexpr (P::kPaged) {
      const int page = __builtin_amdgcn_readlane(pages, (kb - k_lo) / KB - page0);
      return key_off<D>(p, b, hkv, kb, page) * 2;
    } else {
      return static_cast<int64_t>(kb) * (D * 2);
    }
  };
  auto block_bytes = [&](int kb) { return min(k_hi - kb, KB) * (D * 2); };
  // K block -> stage st: thread tid's load i fills row i * KR + tid / KROW, granule tid % KROW, with granule
  // (tid % KROW) ^ (row & 7) of the block (the swizzle does not depend on i)
  constexpr int KR = NT / KROW;
  static_assert(KR % 8 == 0 && 8 % (64 / KROW) == 0, "the swizzle of a granule must not depend on the load, nor its pad on the lane");
  const int k_row0 = tid / KROW;
  const uint32_t k_off = k_row0 * (D * 2) + (((tid % KROW) ^ (k_row0 & 7)) * 16);
  // LDS address of the wave's 1 KB slice of load 0 in stage 0
  const uint32_t k_lds = __builtin_amdgcn_readfirstlane(
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem)) + wave * 1024 + wave * (64 / KROW) / 8 * K_PAD);
  auto k_dma = [&](int64_t off, int bytes, int st, int i) {  // the block's bytes from load i's first row on
    constexpr int kLoad = KR * D * 2;
    lds_dma16(buf_words(kc_head + off + i * kLoad, max(bytes - i * kLoad, 0)), k_off,
              k_lds + st * KSTAGE + i * (NT * 16 + KR / 8 * K_PAD));
  };
  // V block -> registers: pair i is key quad tid % 16 (4 rows) x d octet i * NT / 16 + tid / 16
  const int v_kq = tid % (KB / 4), v_dq = tid / (KB / 4);
  const uint32_t v_off = 4 * v_kq * (D * 2) + v_dq * 16;
  u32x4 vr[VPAIRS][4];
  auto v_load = [&](__amdgpu_buffer_rsrc_t rsrc, int i, int e) {
    vr[i][e] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, v_off + e * (D * 2) + i * NT, 0, 0);
  };
  // registers -> Vt stage st: for each of the octet's 8 d, the quad's 4 keys as one 8-byte write
  const int v_pos = 32 * (v_kq >> 3) + 8 * (v_kq & 3) + 4 * ((v_kq >> 2) & 1);
  const int v_gran = v_pos >> 3, v_half = v_pos & 7;  // the position's granule and offset in it
  // byte offset of d row 8 v_dq's piece; row + c is at (this ^ (c << 4)) + c rows (a row's 128 bytes are aligned)
  const int v_at = 2 * KSTAGE + 8 * v_dq * (VTP * 2) + 16 * v_gran + 2 * v_half;
  auto v_store = [&](int st, int i, int m) {  // d rows 8 (v_dq + i NT / 16) + 2m, + 2m + 1 (d & 7 = 2m, 2m + 1)
    const int at = v_at + st * VSTAGE + i * (NT / 2) * (VTP * 2);
    const uint32_t k0 = vr[i][0][m], k1 = vr[i][1][m], k2 = vr[i][2][m], k3 = vr[i][3][m];
    // byte permutes: the low (0x05040100) and the high (0x07060302) halves of two keys' words
    const u32x2 even = {__builtin_amdgcn_perm(k1, k0, 0x05040100u), __builtin_amdgcn_perm(k3, k2, 0x05040100u)};
    const u32x2 odd = {__builtin_amdgcn_perm(k1, k0, 0x07060302u), __builtin_amdgcn_perm(k3, k2, 0x07060302u)};
    *reinterpret_cast<u32x2*>(smem + (at ^ (2 * m << 4)) + (2 * m) * (VTP * 2)) = even;
    *reinterpret_cast<u32x2*>(smem + (at ^ ((2 * m + 1) << 4)) + (2 * m + 1) * (VTP * 2)) = odd;
  };

  // a wave may see no key of a row in its range: the running max starts at a
  // finite value, so that exp2 of a masked score is 0 and not exp2(-inf + inf)
  float m[2] = {-FLT_MAX, -FLT_MAX}, l[2] = {0.0f, 0.0f};
  f32x4 o[2][NJ];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt)
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[rt][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // K fragment (tile kt, k-step s) of lane (r, q): row 16 kt + r (16 rows and two pads a tile), granule (4s + q) ^ (r & 7)
  // = 8 (s >> 1) + 4 ((s & 1) ^ x2) + (q ^ x01) with x = r & 7: one base for even s, one for odd,
  // each plus 64 (s & ~1) bytes
  const int x2 = (lr >> 2) & 1, y01 = lq ^ (lr & 3);
  constexpr int KTILE = 16 * D * 2 + 2 * K_PAD;
  const int kf0 = KTW * kh * KTILE + lr * (D * 2) + (lr >> 3) * K_PAD;
  const int kfe = kf0 + (4 * x2 + y01) * 16, kfo = kf0 + (4 * (x2 ^ 1) + y01) * 16;
  // V^T fragment (j, ks) of lane (r, q): d row 16 j + r, positions 32 ks + 8q .., granule (4 ks + q) ^ (r & 7)
  const int vfo0 = lr * (VTP * 2) + (4 * (x2 ^ (KG == 2 ? kh : 0)) + y01) * 16;
  const int vfo1 = lr * (VTP * 2) + (4 * (x2 ^ 1) + y01) * 16;

  // Every wave's LDS writes and direct loads are visible to the others.  The 4 VPAIRS loads of V issued after
  // the direct loads may stay in flight (they go to this thread's registers).
  auto publish = [&]() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(4 * VPAIRS) : "memory");
  };
  if (P::kPaged && nblk == 0) {
    find_rows();
    __syncthreads();
  }
  if (nblk > 0) {
    if constexpr (P::kPaged) load_pages(0);
    const int nb = block_bytes(k_lo);
    const int k1 = nblk > 1 ? k_lo + KB : k_lo;
    const int64_t off0 = step_off(k_lo);
    const __amdgpu_buffer_rsrc_t vrs = buf_rsrc(vc_head + off0, nb);
    const __amdgpu_buffer_rsrc_t vrs1 = buf_rsrc(vc_head + step_off(k1), block_bytes(k1));
#pragma unroll
    for (int i = 0; i < KDMA; ++i) k_dma(off0, nb, 0, i);
#pragma unroll
    for (int i = 0; i < VPAIRS; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v_load(vrs, i, e);
    }
    if constexpr (P::kPaged) {  // behind the first keys' loads: one latency for both
      find_rows();
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
      load_q();
    }
#pragma unroll
    for (int i = 0; i < VPAIRS; ++i) {
#pragma unroll
      for (int m4 = 0; m4 < 4; ++m4) v_store(0, i, m4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v_load(vrs1, i, e);
    }
  }
  for (int blk = 0; blk < nblk; ++blk) {
    const int kb = k_lo + KB * blk, st = blk & 1;
    publish();  // block blk is in LDS, stage st ^ 1 is free
    // K of the next block goes in during S^T; its V (in registers since the last iteration) is stored,
    // transposed, during O^T, and the registers take the block after it.  Past the end the loads re-read the
    // last block (never used), so that none sits behind a branch.
    const int kb1 = blk + 1 < nblk ? kb + KB : kb, kb2 = blk + 2 < nblk ? kb + 2 * KB : kb1;
    // (the paged form reads nothing past the end: its descriptors there are empty)
    const int nb1 = P::kPaged && blk + 1 >= nblk ? 0 : block_bytes(kb1);
    if constexpr (P::kPaged) {
      if (blk - page0 >= 32) load_pages(blk);  // steps blk + 1 and blk + 2 are always among the lanes'
    }
    const int64_t off1 = step_off(kb1);
    const __amdgpu_buffer_rsrc_t vrs =
        buf_rsrc(vc_head + step_off(kb2), P::kPaged && blk + 2 >= nblk ? 0 : block_bytes(kb2));

    // S^T = K Q^T: lane (r, q) holds keys 16 kt + 4q + i of row r, for both row tiles
    const unsigned char* Ks = smem + st * KSTAGE;
    auto k_frag = [&](int s, int kt) {
      return *reinterpret_cast<const bf16x8*>(Ks + ((s & 1) ? kfo : kfe) + kt * KTILE + (s & ~1) * 64);
    };
    f32x4 sc[2][KTW];
#pragma unroll
    for (int kt = 0; kt < KTW; ++kt) sc[0][kt] = sc[1][kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // fragments f = (k-step f / KTW, tile f % KTW), KPF of them in flight
    constexpr int KPF = KG == 2 ? 3 : 4;
    bf16x8 kf[KPF], ql[2];
#pragma unroll
    for (int f = 0; f < KPF; ++f) kf[f] = k_frag(f / KTW, f % KTW);
    if constexpr (QL > 0) {
      ql[0] = *q_lds(0, 0);
      ql[1] = *q_lds(1, 0);
    }
#pragma unroll
    for (int f = 0; f < NS * KTW; ++f) {
      const int s = f / KTW, kt = f % KTW;
      const bf16x8 a = kf[f % KPF];
      if (f + KPF < NS * KTW) kf[f % KPF] = k_frag((f + KPF) / KTW, (f + KPF) % KTW);
      if (kt == 0 && s < KDMA) k_dma(off1, nb1, st ^ 1, s);
      const int slot = q_slot(QL, s), reg = slot < 0 ? q_reg(QL, s) : 0;
      sc[0][kt] = mfma16(a, slot < 0 ? qf[0][reg] : ql[0], sc[0][kt]);
      sc[1][kt] = mfma16(a, slot < 0 ? qf[1][reg] : ql[1], sc[1][kt]);
      if (slot >= 0 && slot + 1 < QL && kt == KTW - 1) {  // the next of them
        ql[0] = *q_lds(0, slot + 1);
        ql[1] = *q_lds(1, slot + 1);
      }
    }
    // issue order: fragment f + KPF read ahead of fragment f's two products
    __builtin_amdgcn_sched_group_barrier(0x100, KPF + (QL > 0 ? 2 : 0), 0);
#pragma unroll
    for (int f = 0; f < NS * KTW; ++f) {
      if (f + KPF < NS * KTW) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      const int slot = q_slot(QL, f / KTW);
      if (slot >= 0 && slot + 1 < QL && f % KTW == KTW - 1) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // q
    }

    if (kb + KB > k_free) {
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int kt = 0; kt < KTW; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = kb + 16 * (KTW * kh + kt) + 4 * lq + i;
            if (!(key <= kmax[rt] && key < k_hi)) sc[rt][kt][i] = -INFINITY;
          }
    }
    float mb[2];
    bool grow = false;
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      float x = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < KTW; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) x = fmaxf(x, sc[rt][kt][i]);
      mb[rt] = rows_max(x) * p.scale_log2;
      grow |= mb[rt] > m[rt] + 8.0f;
    }
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        const float m_new = fmaxf(m[rt], mb[rt]);
        const float alpha = __builtin_amdgcn_exp2f(m[rt] - m_new);
        m[rt] = m_new;
        l[rt] *= alpha;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[rt][j] *= alpha;
      }
    }
    // P = exp2(s * scale - m) as the B operand of O^T += V^T P^T: k-slots 8q .. 8q+3 are keys
    // 32 ks + 4q + (0..3) (accumulator tile 2 ks), 8q+4 .. 8q+7 are keys 32 ks + 16 + 4q + (0..3)
    bf16x8 pb[2][KSW];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      float ps = 0.0f;
#pragma unroll
      for (int kt = 0; kt < KTW; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[rt][kt][i] = __builtin_amdgcn_exp2f(fmaf(sc[rt][kt][i], p.scale_log2, -m[rt]));
          ps += sc[rt][kt][i];
        }
      l[rt] += ps;
#pragma unroll
      for (int ks = 0; ks < KSW; ++ks)
        pb[rt][ks] = __builtin_bit_cast(
            bf16x8, u32x4{pk_bf16(sc[rt][2 * ks][0], sc[rt][2 * ks][1]), pk_bf16(sc[rt][2 * ks][2], sc[rt][2 * ks][3]),
                          pk_bf16(sc[rt][2 * ks + 1][0], sc[rt][2 * ks + 1][1]),
                          pk_bf16(sc[rt][2 * ks + 1][2], sc[rt][2 * ks + 1][3])});
    }

    // O^T += V^T P^T
    const unsigned char* Vt = smem + 2 * KSTAGE + st * VSTAGE;
    constexpr int NF = KSW * NJ;  // V^T fragments per block: (ks, j) = (f / NJ, f % NJ)
    constexpr int VPF = 4;        // fragments in flight
    auto v_frag = [&](int f) {
      return *reinterpret_cast<const bf16x8*>(Vt + (f / NJ ? vfo1 : vfo0) + (f % NJ) * 16 * (VTP * 2));
    };
    bf16x8 vf[VPF];
#pragma unroll
    for (int f = 0; f < VPF; ++f) vf[f] = v_frag(f);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const bf16x8 a = vf[f % VPF];
      if (f + VPF < NF) vf[f % VPF] = v_frag(f + VPF);
      const int j = f % NJ, ks = f / NJ;
      o[0][j] = mfma16(a, pb[0][ks], o[0][j]);
      o[1][j] = mfma16(a, pb[1][ks], o[1][j]);
      // the next block's V into the free stage
      constexpr int VST = NF / (4 * VPAIRS);  // fragments per transposed store
      if (f % VST == VST - 1) {
        v_store(st ^ 1, f / VST / 4, (f / VST) % 4);
        if ((f / VST) % 4 == 3) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v_load(vrs, f / VST / 4, e);
        }
      }
    }
    // issue order: fragment f + VPF read ahead of fragment f's two products
    __builtin_amdgcn_sched_group_barrier(0x100, VPF, 1);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      if (f + VPF < NF) __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 1);
    }
  }

  __builtin_amdgcn_s_waitcnt(0);  // no direct load may land in LDS after this
  float lt[2] = {rows_sum(l[0]), rows_sum(l[1])};
  // row tile rt's state (lane (r, q): O[row r][16 j + 4 q + i]) to the output, or to the split's partials
  auto store_tile = [&](auto rtc) {
    constexpr int rt = decltype(rtc)::value;
    if constexpr (P::kPaged) {
      const int r = 32 * rg + 16 * rt + lr;
      if (row_out[r] < 0) return;
      if (row_kmax[r] >= 0) {
        store_row<D, NJ, 16>(p, row_out[r], 4 * lq, o[rt], lt[rt]);
      } else {  // a padded token
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          *reinterpret_cast<u32x2*>(p.out + static_cast<int64_t>(row_out[r]) * D + 16 * j + 4 * lq) = u32x2{0u, 0u};
      }
      return;
    }
    const int r = row0 + 32 * rg + 16 * rt + lr;
    if (r >= n_rows) return;
    const RowAt at = row_at(p, b, hkv, g, r);
    if (p.n_split == 1) {
      const float inv_l = 1.0f / lt[rt];  // (l = 0: every score is -inf, whose softmax is NaN)
#pragma unroll
      for (int j = 0; j < NJ; ++j) store_out4<D>(p, b, at.t, at.hq, 16 * j + 4 * lq, o[rt][j], inv_l);
      return;
    }
    const int64_t pr = part_row(p, b, hkv, r) + split;
    const int64_t n_part = static_cast<int64_t>(p.B) * p.Hkv * p.rows_pad * p.n_split;
    if (lq == 0) {
      p.part[n_part * D + pr] = m[rt];
      p.part[n_part * (D + 1) + pr] = lt[rt];
    }
    if (nblk == 0) return;  // the combine does not use the O of a range without keys (l = 0)
#pragma unroll
    for (int j = 0; j < NJ; ++j) *reinterpret_cast<f32x4*>(p.part + pr * D + 16 * j + 4 * lq) = o[rt][j];
  };
  // The paged form's partial results go out in whole rows, through the wave's 64 D bytes of LDS at `buf`: the
  // accumulators' own layout would write 64 bytes of a row at a time (128 rows of 256: 4.5 us, this way 2.7).
  auto store_part = [&](auto rtc, unsigned char* buf) {
    constexpr int rt = decltype(rtc)::value;
    constexpr int G = D / 4;  // 16-byte granules of a row, XOR-swizzled by the row
    const int r = 32 * rg + 16 * rt + lr;
    const bool ok = row_kmax[r] >= 0;
    const int64_t pr = static_cast<int64_t>(row_part[r]) * p.n_split + split_at(p, split);
    if (ok && lq == 0) {
      const int64_t n_part = static_cast<int64_t>(p.B) * p.Hkv * p.rows_pad * p.n_split;
      p.part[n_part * D + pr] = m[rt];
      p.part[n_part * (D + 1) + pr] = lt[rt];
    }
    if (nblk == 0) return;  // the combine does not use the O of a range without keys (l = 0)
    f32x4* cell = reinterpret_cast<f32x4*>(buf);
#pragma unroll
    for (int j = 0; j < NJ; ++j) cell[lr * G + ((4 * j + lq) ^ lr)] = o[rt][j];
    const uint32_t rows = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(ok));
    auto to = [&](int n) {  // lane n's row
      const int64_t at = static_cast<int64_t>(__builtin_amdgcn_readlane(static_cast<int>(pr >> 32), n)) << 32 |
                         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(pr), n));
      return p.part + at * D;
    };
    if constexpr (G == 64) {
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        const f32x4 x = cell[n * G + (lane ^ n)];
        if ((rows >> n) & 1) *reinterpret_cast<f32x4*>(to(n) + 4 * lane) = x;
      }
    } else {
      static_assert(G == 32, "two rows at a time");
      const int hi = lane >> 5, col = lane & 31;
#pragma unroll
      for (int n = 0; n < 16; n += 2) {
        const f32x4 x = cell[(n + hi) * G + (col ^ (n + hi))];
        float* row = hi ? to(n + 1) : to(n);
        if ((rows >> (n + hi)) & 1) *reinterpret_cast<f32x4*>(row + 4 * col) = x;
      }
    }
  };
  if constexpr (KG == 1) {
    if (P::kPaged && p.n_split > 1) {
      __syncthreads();  // the stages are free
      store_part(std::integral_constant<int, 0>{}, smem + wave * 64 * D);
      store_part(std::integral_constant<int, 1>{}, smem + wave * 64 * D);
      return;
    }
    store_tile(std::integral_constant<int, 0>{});
    store_tile(std::integral_constant<int, 1>{});
  } else {
    // the two waves of a row group merge: wave kh finishes row tile kh, and
    // hands its state of the other tile over in LDS (the K / V stages are free)
    float* xo = reinterpret_cast<float*>(smem);  // [8 waves][NJ][64 lanes][4]
    float* xml = xo + 8 * NJ * 256;              // [8 waves][2][64 lanes]
    static_assert(8 * NJ * 256 * 4 <= 2 * (KSTAGE + VSTAGE), "the exchange must fit in the stages");
    __syncthreads();
    auto hand_over = [&](auto rtc) {
      constexpr int rt = decltype(rtc)::value;
#pragma unroll
      for (int j = 0; j < NJ; ++j) *reinterpret_cast<f32x4*>(xo + ((wave * NJ + j) * 64 + lane) * 4) = o[rt][j];
      xml[wave * 128 + lane] = m[rt];
      xml[wave * 128 + 64 + lane] = lt[rt];
    };
    auto finish = [&](auto rtc) {
      constexpr int rt = decltype(rtc)::value;
      const int w = wave ^ 4;
      const float m2 = xml[w * 128 + lane], l2 = xml[w * 128 + 64 + lane];
      const float mm = fmaxf(m[rt], m2);
      const float a1 = __builtin_amdgcn_exp2f(m[rt] - mm), a2 = __builtin_amdgcn_exp2f(m2 - mm);
      m[rt] = mm;
      lt[rt] = a1 * lt[rt] + a2 * l2;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        o[rt][j] = a1 * o[rt][j] + a2 * *reinterpret_cast<const f32x4*>(xo + ((w * NJ + j) * 64 + lane) * 4);
      if (P::kPaged && p.n_split > 1) store_part(rtc, smem + w * NJ * 1024);  // over what it has just read
      else store_tile(rtc);
    };
    if (kh == 0) hand_over(std::integral_constant<int, 1>{});
    else hand_over(std::integral_constant<int, 0>{});
    __syncthreads();
    if (kh == 0) finish(std::integral_constant<int, 0>{});
    else finish(std::integral_constant<int, 1>{});
  }
}

template <int D, int KG>
__global__ __launch_bounds__(256 * KG) void attn_prefill_kernel(const AttnParams p) {
  __shared__ __align__(128) unsigned char smem[tile_lds<D, KG, AttnParams>()];
  const int n_rb = gridDim.x / p.Hkv;
  // longest key ranges first
  attn_tile<D, KG>(p, smem, blockIdx.z, blockIdx.x % p.Hkv, n_rb - 1 - static_cast<int>(blockIdx.x) / p.Hkv, blockIdx.y);
}

// One wave per (row, kv-head, batch row): the split partials of a row merged.
// A range without keys of the row (l = 0) may have left its O unwritten: it is
// skipped, its loads read the row's first range with keys instead.
// Lane s takes range s's m and l (64 ranges a pass), and eight ranges' O are
// in flight at a time.
template <int D>
__global__ __launch_bounds__(256) void attn_combine_kernel(const AttnParams p) {
  const int lane = threadIdx.x & 63;
  const int g = p.Hq / p.Hkv;
  const int n_rows = p.T * g;
  const int64_t item =
      static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  if (item >= static_cast<int64_t>(p.B) * p.Hkv * n_rows) return;
  const int r = static_cast<int>(item % n_rows);
  const int hkv = static_cast<int>((item / n_rows) % p.Hkv);
  const int b = static_cast<int>(item / (static_cast<int64_t>(n_rows) * p.Hkv));
  const int64_t n_part = static_cast<int64_t>(p.B) * p.Hkv * p.rows_pad * p.n_split;
  const int64_t pr = part_row(p, b, hkv, r);
  const float* pm = p.part + n_part * D + pr;
  const float* pl = p.part + n_part * (D + 1) + pr;
  constexpr int EPL = D / 64, NB = 8;
  typedef float vec __attribute__((ext_vector_type(EPL)));
  vec acc = {};
  float m = -FLT_MAX, lsum = 0.0f;
  for (int s0 = 0; s0 < p.n_split; s0 += 64) {
    const int n = min(64, p.n_split - s0);
    const float ls = lane < n ? pl[s0 + lane] : 0.0f;
    const float ms = lane < n && ls != 0.0f ? pm[s0 + lane] : -FLT_MAX;
    const uint64_t has = __builtin_amdgcn_ballot_w64(ls != 0.0f);
    if (has == 0) continue;
    const int first = __builtin_ctzll(has);
    const float m_new = fmaxf(m, wave_max(ms));
    const float keep = __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    const float w = __builtin_amdgcn_exp2f(ms - m);  // the lane's range
    acc *= keep;
    lsum = lsum * keep + wave_sum(ls != 0.0f ? w * ls : 0.0f);
    for (int s = 0; s < n; s += NB) {
      vec v[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int si = min(s + i, n - 1);
        const int src = (has >> si) & 1 ? si : first;
        v[i] = *reinterpret_cast<const vec*>(p.part + (pr + s0 + src) * D + EPL * lane);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int si = min(s + i, n - 1);
        const float wi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), si));
        if (s + i < n && ((has >> si) & 1)) acc += wi * v[i];  // wave-uniform
      }
    }
  }
  // l = 0: every score is -inf, whose softmax is NaN (zeros in the kernel of fewer rows)
  const float inv_l = n_rows >= kPrefillRows || lsum > 0.0f ? 1.0f / lsum : 0.0f;
  const int t = r / g, hq = hkv * g + r % g;
  if constexpr (EPL == 4) {
    store_out4<D>(p, b, t, hq, EPL * lane, acc, inv_l);
  } else {
    const int64_t bt = static_cast<int64_t>(b) * p.T + t;
    const int64_t row = bt * p.Hq + hq;
    float y0 = acc[0] * inv_l, y1 = acc[1] * inv_l;
    const int d = EPL * lane;
    if (p.qg != nullptr) {
      const uint16_t* gp = p.qg + bt * p.qg_ld + hq * 2 * D + D + d;
      y0 *= sigmoid(bf16_to_f32(gp[0]));
      y1 *= sigmoid(bf16_to_f32(gp[1]));
    }
    *reinterpret_cast<uint32_t*>(p.out + row * D + d) = pk_bf16(y0, y1);
  }
}

}  // namespace
