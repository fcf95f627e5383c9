// Full-attention layers of the hybrid trunk and of the MTP draft head
// (Qwen3.5 gated attention) on gfx950.
//
//   attn_qk_kernel       one wave per token and group of heads: RMSNorm of q and k over
//                        the head dim (y = x / rms(x) * w), the rotary
//                        embedding of the first `rot` dims (rotate-half form,
//                        angle pos * base^(-2i/rot)), q to [B, T, Hq, D]; k and
//                        v appended to the KV cache [B, Hkv, cap, D] at
//                        positions pos0[b] .. pos0[b] + T - 1.
//   attn_fwd_kernel      causal GQA attention over the cache on bf16 MFMA
//                        with an online softmax in fp32.  The query rows of
//                        one kv-head are (token, q-head of its group) pairs,
//                        so the g = Hq / Hkv heads of a group share every K/V
//                        block a workgroup stages in LDS.  RT = 4: four waves
//                        own 16 rows each and walk the same 64-key blocks
//                        (prefill); RT = 1: one 16-row tile, each wave takes
//                        16 keys of every block (decode and draft verify,
//                        where a group has at most 16 rows), and the four
//                        partial softmax states merge in LDS at the end.
//                        Keys may also be split over workgroups; the partial
//                        states then go to a workspace and
//   attn_combine_kernel  merges them.
//   attn_prefill_kernel  long prefills (>= 512 rows per kv-head): 128-row
//                        workgroups, 64-key K / V blocks double-buffered in
//                        LDS (K by direct loads, V transposed on its way in),
//                        one barrier per block; keys split likewise.
//                        The output is multiplied by sigmoid(gate) on the way
//                        out when a gate is given.
//   rms_norm_kernel      the layers' RMSNorm over the hidden size, optionally of
//                        a residual sum it also writes out.
//   pos_add_kernel       the cache offsets' advance and rollback.
//   silu_mul_kernel      the MLP's silu(gate) * up.
#include "gdn_attention.hpp"

namespace {

// ------------------------------------------------------------ attn_qk

struct QkParams {
  const uint16_t* qg;  // [B, T, Hq, 2D]: q, then the output gate, per head (token stride qg_ld)
  const uint16_t* kn;  // [B, T, Hkv, D] (token stride kv_ld)
  const uint16_t* vn;  // [B, T, Hkv, D] (token stride kv_ld)
  int64_t qg_ld, kv_ld;
  const void* qw;      // [D] q_norm weight
  const void* kw;      // [D] k_norm weight
  int wdt;
  const int32_t* pos0;  // [B] position of each row's first new token (its cache length)
  uint16_t* q;          // [B, T, Hq, D]
  uint16_t* kc;         // [B, Hkv, cap, D]
  uint16_t* vc;
  int B, T, Hq, Hkv, cap, rot;
  float eps, log2_base;
};

// One wave takes NH heads of one token (q heads, then k, then v), the last
// wave of a token the rest.  The rotary angles depend on the token and the
// lane only, so exp2 and sincos -- most of the arithmetic, computed per head
// it bounded the kernel at 70.6 us for 4096 tokens of 16 + 2 x 4 heads --
// run once for the NH heads, whose rows are all loaded before the first is
// used and whose chains overlap.  A wave with more heads runs longer, so calls
// of few rows (tokens x heads) take few heads a wave (graph-replayed, us, NH =
// 1 / 3 / 6; a wave per head with the angles of its own before them):
//   16 + 2 x 4 heads of 256:   1 token 3.3, 3.5 / 4.3 / 5.5;  160 tokens (3840 rows) 5.4, 5.0 / 5.2 / 5.9;
//      200 (4800) 5.9, 5.5 / 5.3 / 6.0;  600 (14400) 12.3, 11.0 / 7.9 / 8.0;  700 (16800) 13.7, 12.3 / 8.8 / 8.2;
//      2048 34.1, 29.1 / 17.1 / 16.2
//   4 + 2 x 1 of 256:        600 tokens (3600) 5.2, 4.9 / 5.1 / 5.8;  700 (4200) 5.8, 5.5 / 5.2 / 5.9
//   64 + 2 x 8 of 128:   160 tokens (12800) 7.5, 7.2 / 5.4 / 5.5;  256 (20480) 10.5, 9.9 / 6.6 / 6.4
// (4096 tokens of 16 + 2 x 4 heads of 256, 100 MB, 28.3: 3.6 TB/s).
template <int D, int NH>
__global__ __launch_bounds__(256) void attn_qk_kernel(const QkParams p) {
  constexpr int EPL = D / 64;  // elements per lane
  typedef typename RowVec<EPL>::type vec;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = p.Hq + 2 * p.Hkv;  // q heads, k heads, v heads
  const uint32_t per_tok = (heads + NH - 1) / NH;
  const uint32_t item = blockIdx.x * 4u + wave;
  const uint32_t bt = item / per_tok;
  if (bt >= static_cast<uint32_t>(p.B) * p.T) return;  // wave-uniform
  const int h0 = static_cast<int>(item % per_tok) * NH;
  const int t = static_cast<int>(bt % p.T), b = static_cast<int>(bt / p.T);
  const int d0 = EPL * lane;

  vec raw[NH];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    const int h = min(h0 + n, heads - 1);
    const uint16_t* src;
    if (h < p.Hq) src = p.qg + bt * p.qg_ld + h * 2 * D;
    else if (h < p.Hq + p.Hkv) src = p.kn + bt * p.kv_ld + (h - p.Hq) * D;
    else src = p.vn + bt * p.kv_ld + (h - p.Hq - p.Hkv) * D;
    raw[n] = *reinterpret_cast<const vec*>(src + d0);
  }
  // norm weights as raw bits (converted after every load is issued); a single
  // head's wave loads its own kind's only
  uint32_t qwr[EPL], kwr[EPL];
  const void* qwp = NH > 1 || h0 < p.Hq ? p.qw : p.kw;
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    if (p.wdt == GDN_DTYPE_F32) {
      qwr[e] = static_cast<const uint32_t*>(qwp)[d0 + e];
      if (NH > 1) kwr[e] = static_cast<const uint32_t*>(p.kw)[d0 + e];
    } else {
      qwr[e] = static_cast<const uint16_t*>(qwp)[d0 + e];
      if (NH > 1) kwr[e] = static_cast<const uint16_t*>(p.kw)[d0 + e];
    }
  }
  const int pos = first_pos(p.pos0, b, p.T, p.cap) + t;

  // rotary embedding of dims [0, rot): d < half pairs with d + half
  const int half = p.rot / 2;
  const int shift = half / EPL;  // lanes between partners
  const bool lower = d0 < half;
  const int partner = lower ? lane + shift : lane - shift;
  float sn[EPL], cs[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    sn[e] = 0.0f;
    cs[e] = 1.0f;
  }
  if (d0 < p.rot && h0 < p.Hq + p.Hkv) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const int i = half > 0 ? (d0 + e) % half : 0;
      const float inv_freq = exp2f(-2.0f * static_cast<float>(i) / static_cast<float>(p.rot) * p.log2_base);
      sincosf(static_cast<float>(pos) * inv_freq, &sn[e], &cs[e]);
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
    qw[e] = weight(qwr[e]);
    kw[e] = NH > 1 ? weight(kwr[e]) : qw[e];
  }

  // the heads' chains (sum, norm, exchange) carry no branch, so they overlap
  float r[NH];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const float x = bf16_to_f32(raw[n][e]);
      ss += x * x;
    }
    r[n] = rsqrtf(wave_sum(ss) / D + p.eps);
  }
  vec out[NH];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      // RMSNorm, rounded to bf16 (the norm's output dtype)
      const float x = bf16_to_f32(f32_to_bf16(bf16_to_f32(raw[n][e]) * r[n] * (h0 + n < p.Hq ? qw[e] : kw[e])));
      const float other = __shfl(x, partner, 64);
      const float y = d0 < p.rot ? (lower ? x * cs[e] - other * sn[e] : x * cs[e] + other * sn[e]) : x;
      out[n][e] = f32_to_bf16(y);
    }
  }
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    const int h = h0 + n;
    if (h >= heads) return;  // wave-uniform
    if (h < p.Hq) {
      *reinterpret_cast<vec*>(p.q + (static_cast<int64_t>(bt) * p.Hq + h) * D + d0) = out[n];
    } else {
      const bool is_k = h < p.Hq + p.Hkv;  // v goes into the cache as is
      const int hkv = h - p.Hq - (is_k ? 0 : p.Hkv);
      *reinterpret_cast<vec*>((is_k ? p.kc : p.vc) + ((static_cast<int64_t>(b) * p.Hkv + hkv) * p.cap + pos) * D + d0) =
          is_k ? out[n] : raw[n];
    }
  }
}

// ------------------------------------------------------------ rms_norm

// Eight weights from index i (a multiple of 8) as floats: one 16-byte load for
// bf16 / fp16, two for fp32 (the branch is uniform).
__device__ __forceinline__ void load_w8(const void* w, int wdt, int i, float out[8]) {
  if (wdt == GDN_DTYPE_F32) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(static_cast<const float*>(w) + i);
    const f32x4 b = *reinterpret_cast<const f32x4*>(static_cast<const float*>(w) + i + 4);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      out[k] = a[k];
      out[4 + k] = b[k];
    }
  } else {
    const u32x4 v = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(w) + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint16_t lo = static_cast<uint16_t>(v[k] & 0xffffu), hi = static_cast<uint16_t>(v[k] >> 16);
      out[2 * k] = wdt == GDN_DTYPE_BF16 ? bf16_to_f32(lo) : f16_to_f32(lo);
      out[2 * k + 1] = wdt == GDN_DTYPE_BF16 ? bf16_to_f32(hi) : f16_to_f32(hi);
    }
  }
}

// One workgroup per row; 8 bf16 elements per thread and chunk, chunk c of
// thread t at 8 t + 2048 c.  With a residual, the row is h = bf16(x + res)
// (written to h_out when given) and y = norm(h); y's rows are y_ld elements
// apart.  The first kRegChunks chunks of h stay in registers between the sum
// of squares and the output (one pass over memory up to D = 8192); chunks
// beyond are read again, from h_out when this thread wrote them (h_out may
// alias x), else recomputed.
constexpr int kRegChunks = 4;
__global__ __launch_bounds__(256) void rms_norm_kernel(const uint16_t* x, const uint16_t* res, uint16_t* h_out,
                                                       const void* w, int wdt, uint16_t* y, int64_t y_ld, int D,
                                                       float eps) {
  const int64_t row = blockIdx.x;
  const uint16_t* xr = x + row * D;
  const uint16_t* rr = res != nullptr ? res + row * D : nullptr;
  auto load_h = [&](int c) {
    u32x4 v = *reinterpret_cast<const u32x4*>(xr + c);
    if (rr != nullptr) {
      const u32x4 r = *reinterpret_cast<const u32x4*>(rr + c);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = pk_bf16(__uint_as_float(v[k] << 16) + __uint_as_float(r[k] << 16),
                       __uint_as_float(v[k] & 0xffff0000u) + __uint_as_float(r[k] & 0xffff0000u));
    }
    return v;
  };
  auto sq = [](u32x4 v) {
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = __uint_as_float(v[k] << 16), bb = __uint_as_float(v[k] & 0xffff0000u);
      ss += a * a + bb * bb;
    }
    return ss;
  };
  const int c0 = 8 * threadIdx.x;
  u32x4 hv[kRegChunks];
  float wv[kRegChunks][8];
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < kRegChunks; ++j) {
    const int c = c0 + 2048 * j;
    if (c < D) {
      hv[j] = load_h(c);
      load_w8(w, wdt, c, wv[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kRegChunks; ++j) {
    const int c = c0 + 2048 * j;
    if (c < D) {
      if (h_out != nullptr) *reinterpret_cast<u32x4*>(h_out + row * D + c) = hv[j];
      ss += sq(hv[j]);
    }
  }
  for (int c = c0 + 2048 * kRegChunks; c < D; c += 2048) {
    const u32x4 v = load_h(c);
    if (h_out != nullptr) *reinterpret_cast<u32x4*>(h_out + row * D + c) = v;
    ss += sq(v);
  }
  __shared__ float part[4];
  ss = wave_sum(ss);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
  __syncthreads();
  const float r = rsqrtf((part[0] + part[1] + part[2] + part[3]) / D + eps);
  auto out8 = [&](int c, u32x4 v, const float* wk) {
    u32x4 o;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      o[k] = pk_bf16(__uint_as_float(v[k] << 16) * r * wk[2 * k], __uint_as_float(v[k] & 0xffff0000u) * r * wk[2 * k + 1]);
    *reinterpret_cast<u32x4*>(y + row * y_ld + c) = o;
  };
#pragma unroll
  for (int j = 0; j < kRegChunks; ++j) {
    const int c = c0 + 2048 * j;
    if (c < D) out8(c, hv[j], wv[j]);
  }
  for (int c = c0 + 2048 * kRegChunks; c < D; c += 2048) {
    const u32x4 v = h_out != nullptr ? *reinterpret_cast<const u32x4*>(h_out + row * D + c) : load_h(c);
    float wk[8];
    load_w8(w, wdt, c, wk);
    out8(c, v, wk);
  }
}

// ------------------------------------------------------------ pos_add

// pos[b] = max(pos[b] + delta, lo): a KV cache's advance and rollback, one
// launch each (the rollback was a subtraction and a clamp, two launches of
// 1.5 us and 4 us of host time for a few integers).
__global__ __launch_bounds__(256) void pos_add_kernel(int32_t* pos, int B, int32_t delta, int32_t lo) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < B) pos[b] = max(static_cast<int32_t>(static_cast<uint32_t>(pos[b]) + static_cast<uint32_t>(delta)), lo);
}

// ------------------------------------------------------------ silu_mul

// out[r, i] = silu(gu[r, i]) * gu[r, I + i]; 8 elements per thread.
__global__ __launch_bounds__(256) void silu_mul_kernel(const uint16_t* gu, uint16_t* out, int64_t rows, int I) {
  const int64_t i8 = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8;
  if (i8 >= rows * I) return;
  const int64_t r = i8 / I;
  const int c = static_cast<int>(i8 % I);
  const u32x4 gv = *reinterpret_cast<const u32x4*>(gu + r * 2 * I + c);
  const u32x4 uv = *reinterpret_cast<const u32x4*>(gu + r * 2 * I + I + c);
  u32x4 o;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float g0 = __uint_as_float(gv[k] << 16), g1 = __uint_as_float(gv[k] & 0xffff0000u);
    const float u0 = __uint_as_float(uv[k] << 16), u1 = __uint_as_float(uv[k] & 0xffff0000u);
    o[k] = pk_bf16(silu(g0) * u0, silu(g1) * u1);
  }
  *reinterpret_cast<u32x4*>(out + i8) = o;
}

int64_t attn_rows_pad(int64_t T, int64_t Hq, int64_t Hkv, int rt) {
  const int64_t n_rows = T * (Hq / Hkv);
  const int64_t tile = 16 * rt;
  return (n_rows + tile - 1) / tile * tile;
}

int attn_rt(int64_t T, int64_t Hq, int64_t Hkv) { return T * (Hq / Hkv) <= 16 ? 1 : 4; }

}  // namespace

extern "C" size_t gdn_attn_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                           int64_t n_split) {
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || n_split < 1) return 0;
  if (n_split == 1) return 0;
  const int64_t rows_pad = attn_rows_pad(T, Hq, Hkv, attn_rt(T, Hq, Hkv));
  return static_cast<size_t>(B * Hkv * rows_pad * n_split) * (D + 2) * sizeof(float);
}

extern "C" int gdn_attn_qk(const void* qg, int64_t qg_ld, const void* k_new, const void* v_new, int64_t kv_ld,
                           const void* q_norm_w, const void* k_norm_w, int w_dtype, float eps, const int32_t* pos0,
                           void* q_out, void* k_cache, void* v_cache, int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                           int64_t D, int64_t cap, int64_t rot, float rope_base, void* stream) {
  using gdn_host::fail;
  if (D != 128 && D != 256) return fail(GDN_ERR_UNSUPPORTED, "gdn_attn_qk: head dim must be 128 or 256 (got %lld)", (long long)D);
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || cap < T || cap > INT32_MAX)
    return fail(GDN_ERR_INVALID, "gdn_attn_qk: bad sizes");
  if (rot < 0 || rot > D || rot % (2 * (D / 64)) != 0 || (rot > 0 && (rot / 2) % (D / 64) != 0))
    return fail(GDN_ERR_UNSUPPORTED, "gdn_attn_qk: rotary dims %lld not supported for head dim %lld", (long long)rot,
                (long long)D);
  if (!gdn_host::dtype_ok(w_dtype) || !(rope_base > 0.0f) || !(eps >= 0.0f))
    return fail(GDN_ERR_INVALID, "gdn_attn_qk: bad norm weight dtype, eps or rope base");
  if (B * T == 0) return GDN_OK;
  if (!qg || !k_new || !v_new || !q_norm_w || !k_norm_w || !pos0 || !q_out || !k_cache || !v_cache)
    return fail(GDN_ERR_INVALID, "gdn_attn_qk: null pointer");
  if (B * T * (Hq + 2 * Hkv) > INT32_MAX) return fail(GDN_ERR_UNSUPPORTED, "gdn_attn_qk: problem too large");
  if (qg_ld == 0) qg_ld = 2 * Hq * D;
  if (kv_ld == 0) kv_ld = Hkv * D;
  if (qg_ld < 2 * Hq * D || kv_ld < Hkv * D) return fail(GDN_ERR_INVALID, "gdn_attn_qk: token strides below the rows");
  QkParams p;
  p.qg = static_cast<const uint16_t*>(qg);
  p.kn = static_cast<const uint16_t*>(k_new);
  p.vn = static_cast<const uint16_t*>(v_new);
  p.qg_ld = qg_ld;
  p.kv_ld = kv_ld;
  p.qw = q_norm_w;
  p.kw = k_norm_w;
  p.wdt = w_dtype;
  p.pos0 = pos0;
  p.q = static_cast<uint16_t*>(q_out);
  p.kc = static_cast<uint16_t*>(k_cache);
  p.vc = static_cast<uint16_t*>(v_cache);
  p.B = static_cast<int>(B);
  p.T = static_cast<int>(T);
  p.Hq = static_cast<int>(Hq);
  p.Hkv = static_cast<int>(Hkv);
  p.cap = static_cast<int>(cap);
  p.rot = static_cast<int>(rot);
  p.eps = eps;
  p.log2_base = log2f(rope_base);
  hipStream_t st = static_cast<hipStream_t>(stream);
  // heads per wave by the rows of all heads (attn_qk_kernel's comment has both sides of each line)
  auto launch = [&](auto nh) {
    constexpr int NH = decltype(nh)::value;
    const dim3 grid(static_cast<unsigned>((B * T * ((Hq + 2 * Hkv + NH - 1) / NH) + 3) / 4));
    if (D == 256) hipLaunchKernelGGL((attn_qk_kernel<256, NH>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((attn_qk_kernel<128, NH>), grid, dim3(256), 0, st, p);
  };
  const int64_t rows = B * T * (Hq + 2 * Hkv);
  if (rows <= 4096) launch(std::integral_constant<int, 1>{});
  else if (rows <= 16384) launch(std::integral_constant<int, 3>{});
  else launch(std::integral_constant<int, 6>{});
  return gdn_host::check_launch("gdn_attn_qk");
}

extern "C" int gdn_attn_fwd(const void* q, const void* qg, int64_t qg_ld, const void* k_cache, const void* v_cache,
                            const int32_t* pos0, void* out, float scale, int64_t B, int64_t T, int64_t Hq,
                            int64_t Hkv, int64_t D, int64_t cap, int64_t kv_len_max, int64_t n_split,
                            void* workspace, size_t workspace_bytes, void* stream) {
  using gdn_host::fail;
  if (D != 128 && D != 256) return fail(GDN_ERR_UNSUPPORTED, "gdn_attn_fwd: head dim must be 128 or 256 (got %lld)", (long long)D);
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || cap < T || cap > INT32_MAX || n_split < 1 ||
      n_split > 65535 || kv_len_max < T || kv_len_max > cap)
    return fail(GDN_ERR_INVALID, "gdn_attn_fwd: bad sizes (kv_len_max must lie in [T, cap])");
  if (!(scale > 0.0f)) return fail(GDN_ERR_INVALID, "gdn_attn_fwd: scale must be positive");
  if (B * T == 0) return GDN_OK;
  if (!q || !k_cache || !v_cache || !pos0 || !out) return fail(GDN_ERR_INVALID, "gdn_attn_fwd: null pointer");
  if (qg_ld == 0) qg_ld = 2 * Hq * D;
  if (qg && qg_ld < 2 * Hq * D) return fail(GDN_ERR_INVALID, "gdn_attn_fwd: gate token stride below the row");
  if (!gdn_host::aligned(q, 16) || !gdn_host::aligned(k_cache, 16) || !gdn_host::aligned(v_cache, 16) ||
      !gdn_host::aligned(out, 8) || (qg && (!gdn_host::aligned(qg, 8) || qg_ld % 4 != 0)))
    return fail(GDN_ERR_INVALID, "gdn_attn_fwd: misaligned pointer");
  const int rt = attn_rt(T, Hq, Hkv);
  const int64_t rows_pad = attn_rows_pad(T, Hq, Hkv, rt);
  const int64_t n_rb = rows_pad / (16 * rt);
  if (B > 65535 || Hkv * n_rb > INT32_MAX || B * Hkv * rows_pad * n_split * (D + 2) > (int64_t(1) << 40))
    return fail(GDN_ERR_UNSUPPORTED, "gdn_attn_fwd: problem too large");
  const size_t need = gdn_attn_workspace_bytes(B, T, Hq, Hkv, D, n_split);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !gdn_host::aligned(workspace, 16)))
    return fail(GDN_ERR_INVALID, "gdn_attn_fwd: workspace of %zu bytes is below the %zu needed for %lld splits",
                workspace_bytes, need, (long long)n_split);
  AttnParams p;
  p.q = static_cast<const uint16_t*>(q);
  p.qg = static_cast<const uint16_t*>(qg);
  p.qg_ld = qg_ld;
  p.kc = static_cast<const uint16_t*>(k_cache);
  p.vc = static_cast<const uint16_t*>(v_cache);
  p.pos0 = pos0;
  p.out = static_cast<uint16_t*>(out);
  p.part = static_cast<float*>(workspace);
  p.B = static_cast<int>(B);
  p.T = static_cast<int>(T);
  p.Hq = static_cast<int>(Hq);
  p.Hkv = static_cast<int>(Hkv);
  p.cap = static_cast<int>(cap);
  p.n_split = static_cast<int>(n_split);
  p.split_len = static_cast<int>(((kv_len_max + n_split - 1) / n_split + KB - 1) / KB * KB);
  p.rows_pad = static_cast<int>(rows_pad);
  p.scale_log2 = scale * kLog2e;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (T * (Hq / Hkv) >= kPrefillRows) {
    const int64_t n_prb = (T * (Hq / Hkv) + PR - 1) / PR;
    if (Hkv * n_prb > INT32_MAX) return fail(GDN_ERR_UNSUPPORTED, "gdn_attn_fwd: problem too large");
    const dim3 pgrid(static_cast<unsigned>(Hkv * n_prb), static_cast<unsigned>(n_split), static_cast<unsigned>(B));
    if (D == 256) hipLaunchKernelGGL((attn_prefill_kernel<256, 2>), pgrid, dim3(512), 0, st, p);
    else hipLaunchKernelGGL((attn_prefill_kernel<128, 1>), pgrid, dim3(256), 0, st, p);
  } else if (const dim3 grid(static_cast<unsigned>(n_split), static_cast<unsigned>(Hkv * n_rb), static_cast<unsigned>(B));
             D == 256) {
    if (rt == 4) hipLaunchKernelGGL((attn_fwd_kernel<256, 4>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((attn_fwd_kernel<256, 1>), grid, dim3(256), 0, st, p);
  } else {
    if (rt == 4) hipLaunchKernelGGL((attn_fwd_kernel<128, 4>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((attn_fwd_kernel<128, 1>), grid, dim3(256), 0, st, p);
  }
  int rc = gdn_host::check_launch("gdn_attn_fwd");
  if (rc != GDN_OK || n_split == 1) return rc;
  const int64_t waves = B * Hkv * T * (Hq / Hkv);
  const dim3 cgrid(static_cast<unsigned>((waves + 3) / 4));
  if (D == 256) hipLaunchKernelGGL(attn_combine_kernel<256>, cgrid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(attn_combine_kernel<128>, cgrid, dim3(256), 0, st, p);
  return gdn_host::check_launch("gdn_attn_fwd/combine");
}

extern "C" int gdn_rms_norm(const void* x, const void* res, void* h_out, const void* w, int w_dtype, void* y,
                            int64_t y_ld, int64_t rows, int64_t D, float eps, void* stream) {
  using gdn_host::fail;
  if (rows < 0 || D <= 0 || D % 8 != 0 || D > INT32_MAX || rows > INT32_MAX)
    return fail(GDN_ERR_INVALID, "gdn_rms_norm: bad sizes (D must be a multiple of 8)");
  if (y_ld == 0) y_ld = D;
  if (y_ld < D || y_ld % 8 != 0) return fail(GDN_ERR_INVALID, "gdn_rms_norm: y row stride must be >= D and a multiple of 8");
  if (!gdn_host::dtype_ok(w_dtype) || !(eps >= 0.0f)) return fail(GDN_ERR_INVALID, "gdn_rms_norm: bad weight dtype or eps");
  if (rows == 0) return GDN_OK;
  if (!x || !w || !y) return fail(GDN_ERR_INVALID, "gdn_rms_norm: null pointer");
  if (!gdn_host::aligned(x, 16) || !gdn_host::aligned(y, 16) || !gdn_host::aligned(w, 16) ||
      (res && !gdn_host::aligned(res, 16)) || (h_out && !gdn_host::aligned(h_out, 16)))
    return fail(GDN_ERR_INVALID, "gdn_rms_norm: misaligned pointer");
  hipLaunchKernelGGL(rms_norm_kernel, dim3(static_cast<unsigned>(rows)), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(res), static_cast<uint16_t*>(h_out),
                     w, w_dtype, static_cast<uint16_t*>(y), y_ld, static_cast<int>(D), eps);
  return gdn_host::check_launch("gdn_rms_norm");
}

extern "C" int gdn_pos_add(int32_t* pos, int64_t B, int32_t delta, int32_t lo, void* stream) {
  using gdn_host::fail;
  if (B < 0 || B > INT32_MAX) return fail(GDN_ERR_INVALID, "gdn_pos_add: bad sizes");
  if (B == 0) return GDN_OK;
  if (!pos) return fail(GDN_ERR_INVALID, "gdn_pos_add: null pointer");
  hipLaunchKernelGGL(pos_add_kernel, dim3(static_cast<unsigned>((B + 255) / 256)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), pos, static_cast<int>(B), delta, lo);
  return gdn_host::check_launch("gdn_pos_add");
}

extern "C" int gdn_silu_mul(const void* gate_up, void* out, int64_t rows, int64_t I, void* stream) {
  using gdn_host::fail;
  if (rows < 0 || I <= 0 || I % 8 != 0 || I > INT32_MAX) return fail(GDN_ERR_INVALID, "gdn_silu_mul: bad sizes (I must be a multiple of 8)");
  if (rows == 0) return GDN_OK;
  if (!gate_up || !out) return fail(GDN_ERR_INVALID, "gdn_silu_mul: null pointer");
  if (!gdn_host::aligned(gate_up, 16) || !gdn_host::aligned(out, 16)) return fail(GDN_ERR_INVALID, "gdn_silu_mul: misaligned pointer");
  const int64_t n8 = rows * I / 8;
  if ((n8 + 255) / 256 > INT32_MAX) return fail(GDN_ERR_UNSUPPORTED, "gdn_silu_mul: problem too large");
  hipLaunchKernelGGL(silu_mul_kernel, dim3(static_cast<unsigned>((n8 + 255) / 256)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), static_cast<const uint16_t*>(gate_up), static_cast<uint16_t*>(out),
                     rows, static_cast<int>(I));
  return gdn_host::check_launch("gdn_silu_mul");
}
