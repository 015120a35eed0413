// The way into the 4-bit cache and out of it as dense rows (elementwise passes, bound by memory).
//
// Write: q rotated; k rotated, rounded to bf16 and quantised; v quantised.  A lane owns eight neighbouring channels, so a head's row is 8,
// 16 or 32 neighbouring lanes; a group of 64 channels is eight lanes, which agree on its least and greatest value by three shuffles; the
// partner of a channel rotated by halves lies with another lane of the row and comes by shuffle.  A warp stays with one token, whose
// angles a lane then loads once for all of its rows.
//
// Gather: the contexts of a ragged step as dense bf16 rows, for the prompt kernel.
//
// 16384 tokens, 16 heads on 8 of 128: 0.22 GB written and read in 59 us, 3.7 TB/s.  A warp's two loads in a row (position, then angles) and the
// quantising are what it waits for: 45 us without a cache slot, 50 with the angles close by.  17 K tokens unpacked: 0.09 GB in 18 us, 5.0 TB/s.
#include "dtype.cuh"
#include "host_util.cuh"
#include "kv4.cuh"

#include <type_traits>

namespace mvb {

struct Kv4WriteParams {
  const __nv_bfloat16* q;
  __nv_bfloat16* q_out;
  __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t q_stride, qo_stride, k_stride, v_stride;
  const int64_t* positions;
  const float* cos_sin;                // nullptr: nothing is rotated
  int64_t max_pos;
  const int32_t* slots;                // nullptr: nothing is cached
  uint8_t *k_codes, *v_codes;
  uint32_t *k_affine, *v_affine;
  int64_t num_slots;
  FastDiv by_block, by_token;
  int tokens, hq, hkv, block_size, rot, k_in_place;
  int q_warps, k_warps;                // of a token
  int* dev_status;
};

// The codes round(t / s), 0 <= t <= 15 s (1 + 2^-8), of eight channels as a word, r within 2^-22 of 1 / s.  f is the correctly rounded
// quotient: with f0 = t r the remainder t - f0 s takes 8 bits (s has 8) and is exact, f0 + r (t - f0 s) is within 2^-44 of t / s, and no
// such quotient is that near the middle between two fp32 numbers.  So halves are halves and go to the even code.  Adding 1.5 * 2^23 rounds
// to a whole number, which then stands in the float's last bits.
__device__ __forceinline__ uint32_t kv4_codes(const float2 (&t)[4], float s, float r) {
  constexpr float kRound = 12582912.f;
  constexpr uint32_t kPlaces = 0x11111111u;                  // one in each of the eight 4-bit places
  const float2 r2 = make_float2(r, r), minus_s = make_float2(-s, -s), round2 = make_float2(kRound, kRound);
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f0 = mul_f32x2(t[e], r2), f = add_f32x2(fma_f32x2(fma_f32x2(f0, minus_s, t[e]), r2, f0), round2);
    word += (__float_as_uint(f.x) << kv4_shift(2 * e)) + (__float_as_uint(f.y) << kv4_shift(2 * e + 1));
  }
  return word - __float_as_uint(kRound) * kPlaces;           // modulo 2^32: the codes alone remain
}

// (what is not a number stays so: it has to reach the scale and the minimum)
__device__ __forceinline__ uint32_t min_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 x = __hmin2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 x = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&x);
}

// A warp works on queries, on keys or on values of its token: `by_token` counts the warps of a token, those of q first, then those of k.
template <int D, bool INTER, int ITEMS>
__global__ void __launch_bounds__(256, ITEMS == 4 ? 4 : 1) kv4_write_kernel(const Kv4WriteParams p) {
  constexpr int LPH = D / 8, RPW = 32 / LPH;                 // lanes of a row, rows a warp holds at once
  constexpr uint32_t FULL = 0xffffffffu;
  const int lane = threadIdx.x & 31, c = lane % LPH, sub = lane / LPH;
  const uint32_t warp = blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint32_t t = p.by_token.div(warp);
  if (t >= static_cast<uint32_t>(p.tokens)) return;          // warp-uniform
  int part = static_cast<int>(warp - t * p.by_token.n);
  const bool is_q = part < p.q_warps;
  if (!is_q) part -= p.q_warps;
  const bool is_v = !is_q && part >= p.k_warps;
  if (is_v) part -= p.k_warps;
  const int heads = is_q ? p.hq : p.hkv, head0 = part * (RPW * ITEMS) + sub;
  const __nv_bfloat16* src = is_q ? p.q + static_cast<int64_t>(t) * p.q_stride
                                  : is_v ? p.v + static_cast<int64_t>(t) * p.v_stride : p.k + static_cast<int64_t>(t) * p.k_stride;
  src += static_cast<int64_t>(head0) * D + c * 8;
  uint4 x[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    x[i] = make_uint4(0, 0, 0, 0);
    if (head0 + i * RPW < heads) x[i] = *reinterpret_cast<const uint4*>(src + i * RPW * D);
  }
  int64_t slot = -1;
  if (!is_q) {
    slot = p.slots[t];
    if (slot < -1 || slot >= p.num_slots) {
      if (lane == 0) report(p.dev_status, kDevBadSlot, t);
      slot = -1;
    }
  }
  if (p.cos_sin != nullptr && !is_v) {
    const int half = p.rot >> 1;
    const bool turns = c * 8 < p.rot;                        // this lane's channels are rotated
    const bool second = !INTER && c * 8 >= half;             // halves: the lane holds the second one of its pairs
    const int partner = sub * LPH + (turns ? (second ? c - half / 8 : c + half / 8) : c);
    const int64_t pos = p.positions[t];
    const bool ok = pos >= 0 && pos < p.max_pos;
    if (!ok && lane == 0) report(p.dev_status, kDevBadPosition, t);
    float cs[8], sn[8];                                      // of the lane's eight channels, the sine with the sign that the channel's product has
    if (turns && ok) {
      const float* tab = p.cos_sin + pos * p.rot + (INTER ? c * 4 : (second ? c * 8 - half : c * 8));
      const float sign = second ? 1.f : -1.f;                // (a sign changes no rounding)
#pragma unroll
      for (int e = 0; e < (INTER ? 4 : 8); e += 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(tab + e)), b = __ldg(reinterpret_cast<const float4*>(tab + half + e));
        const float ca[4] = {a.x, a.y, a.z, a.w}, sa[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (INTER) {
            cs[2 * k] = cs[2 * k + 1] = ca[k];
            sn[2 * k] = -sa[k]; sn[2 * k + 1] = sa[k];
          } else {
            cs[e + k] = ca[k];
            sn[e + k] = sign * sa[k];
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, o[4] = {0, 0, 0, 0};
      if constexpr (!INTER) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __shfl_sync(FULL, w[e], partner);
      }
      if (turns && ok) {
        // own cos +- other sin: two products and a sum, each rounded by itself (the paired instructions would be fused)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = bf16_lo(w[e]), b = bf16_hi(w[e]), other_a = INTER ? b : bf16_lo(o[e]), other_b = INTER ? a : bf16_hi(o[e]);
          w[e] = pack_bf16(__fadd_rn(__fmul_rn(a, cs[2 * e]), __fmul_rn(other_a, sn[2 * e])),
                           __fadd_rn(__fmul_rn(b, cs[2 * e + 1]), __fmul_rn(other_b, sn[2 * e + 1])));
        }
        x[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    if (!is_q && p.k_in_place && turns && ok) {
      __nv_bfloat16* dst = p.k + static_cast<int64_t>(t) * p.k_stride + static_cast<int64_t>(head0) * D + c * 8;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (head0 + i * RPW < heads) *reinterpret_cast<uint4*>(dst + i * RPW * D) = x[i];
    }
  }
  if (is_q) {
    __nv_bfloat16* dst = p.q_out + static_cast<int64_t>(t) * p.qo_stride + static_cast<int64_t>(head0) * D + c * 8;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (head0 + i * RPW < heads) *reinterpret_cast<uint4*>(dst + i * RPW * D) = x[i];
    return;
  }
  if (slot < 0) return;                                      // warp-uniform
  const int64_t block = p.by_block.div(static_cast<uint32_t>(slot));
  const int64_t at = kv4_row(block, p.hkv, head0, p.block_size, static_cast<int>(slot - block * p.block_size));
  uint32_t* codes = reinterpret_cast<uint32_t*>(is_v ? p.v_codes : p.k_codes) + at * (D / 8) + kv4_word<D>(c, !is_v);
  uint32_t* affine = (is_v ? p.v_affine : p.k_affine) + at * (D / 64) + (c >> 3);
  const int64_t code_step = static_cast<int64_t>(RPW) * p.block_size * (D / 8), affine_step = static_cast<int64_t>(RPW) * p.block_size * (D / 64);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    // the group's least and greatest value, as the pair (least, -greatest): one minimum for both; every lane of the warp takes part
    const uint32_t least2 = min_bf16x2(min_bf16x2(x[i].x, x[i].y), min_bf16x2(x[i].z, x[i].w));
    const uint32_t most2 = max_bf16x2(max_bf16x2(x[i].x, x[i].y), max_bf16x2(x[i].z, x[i].w));
    uint32_t pair = min_bf16x2(__byte_perm(least2, most2, 0x5410) ^ 0x80000000u, __byte_perm(least2, most2, 0x7632) ^ 0x80000000u);
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) pair = min_bf16x2(pair, __shfl_xor_sync(FULL, pair, off));
    const float lo = bf16_lo(pair), hi = -bf16_hi(pair);
    const float scale = __bfloat162float(__float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f)));
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    float2 d[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = add_f32x2(make_float2(bf16_lo(w[e]), bf16_hi(w[e])), make_float2(-lo, -lo));
    uint32_t word = 0;
    if (scale > 0x1p-100f && scale < 0x1p100f) {             // the usual case: the reciprocal is a normal number, no code passes 15
      word = kv4_codes(d, scale, fast_rcp(scale));
    } else if (scale > 0.f) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        word |= (static_cast<uint32_t>(fminf(rintf(__fdiv_rn(d[e].x, scale)), 15.f)) & 15u) << kv4_shift(2 * e);
        word |= (static_cast<uint32_t>(fminf(rintf(__fdiv_rn(d[e].y, scale)), 15.f)) & 15u) << kv4_shift(2 * e + 1);
      }
    }
    if (head0 + i * RPW < heads) {
      codes[i * code_step] = word;
      if ((c & 7) == 0) affine[i * affine_step] = pack_bf16(scale, lo);
    }
  }
}

struct Kv4GatherParams {
  const uint32_t *k_codes, *v_codes, *k_affine, *v_affine;
  __nv_bfloat16 *k_out, *v_out;
  const int32_t* cu;
  const int32_t* block_table;
  int64_t table_stride, num_blocks;
  FastDiv by_token, by_block;
  int table_width, num_seqs, rows, hkv, block_size;
  int* dev_status;
};

// A lane takes eight channels of the key and of the value of a head, whose places in the cache differ by the base address only.
template <int D, int ITEMS>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const Kv4GatherParams p) {
  constexpr int LPH = D / 8, RPW = 32 / LPH;
  const int lane = threadIdx.x & 31, c = lane % LPH, sub = lane / LPH;
  const uint32_t warp = blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint32_t t = p.by_token.div(warp);
  if (t >= static_cast<uint32_t>(p.rows)) return;
  const int total = p.cu[p.num_seqs];
  if (static_cast<int>(t) >= total) return;                  // rows behind the last sequence are left as they are
  const int b = seq_of_row(p.cu, p.num_seqs, t);
  const int token = static_cast<int>(t) - p.cu[b];
  const int col = p.by_block.div(max(token, 0));             // (negative: a list of lengths that does not begin at 0)
  const int64_t block = token >= 0 && col < p.table_width ? p.block_table[b * p.table_stride + col] : -1;
  const bool ok = block >= 0 && block < p.num_blocks;
  if (!ok && lane == 0) report(p.dev_status, kDevBadBlock, b);
  const int head0 = static_cast<int>(warp - t * p.by_token.n) * (RPW * ITEMS) + sub;
  const int64_t row = ok ? kv4_row(block, p.hkv, head0, p.block_size, token - col * p.block_size) : 0;
  const uint32_t *kc = p.k_codes + row * (D / 8) + kv4_word<D>(c, true), *vc = p.v_codes + row * (D / 8) + kv4_word<D>(c, false);
  const uint32_t *ka = p.k_affine + row * (D / 64) + (c >> 3), *va = p.v_affine + row * (D / 64) + (c >> 3);
  const int64_t code_step = static_cast<int64_t>(RPW) * p.block_size * (D / 8), affine_step = static_cast<int64_t>(RPW) * p.block_size * (D / 64);
  uint32_t word[ITEMS][2], affine[ITEMS][2];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    word[i][0] = word[i][1] = affine[i][0] = affine[i][1] = 0;           // a bad block reads as zeros
    if (head0 + i * RPW < p.hkv && ok) {
      word[i][0] = __ldg(kc + i * code_step); word[i][1] = __ldg(vc + i * code_step);
      affine[i][0] = __ldg(ka + i * affine_step); affine[i][1] = __ldg(va + i * affine_step);
    }
  }
  const int64_t to = (static_cast<int64_t>(t) * p.hkv + head0) * D + c * 8;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (head0 + i * RPW >= p.hkv) continue;
    float y[8];
    kv4_values(word[i][0], affine[i][0], y);
    store_vec<__nv_bfloat16, 8>(p.k_out + to + i * RPW * D, y);
    kv4_values(word[i][1], affine[i][1], y);
    store_vec<__nv_bfloat16, 8>(p.v_out + to + i * RPW * D, y);
  }
}

template <class F>
static int by_head_dim(int d, F&& f) {
  if (d == 64) return f(std::integral_constant<int, 64>{});
  if (d == 128) return f(std::integral_constant<int, 128>{});
  return f(std::integral_constant<int, 256>{});
}

}  // namespace mvb

extern "C" int mvb_rotary_kv4_write(const void* q, int64_t q_row_stride, void* q_out, int64_t q_out_row_stride, void* k,
                                    int64_t k_row_stride, const void* v, int64_t v_row_stride, const int64_t* positions,
                                    const float* cos_sin, int64_t max_pos, int rotary_dim, int interleaved, const int32_t* slot_mapping,
                                    const mvb_kv4_cache* cache, int num_tokens, int num_q_heads, int k_in_place, int32_t* dev_status,
                                    void* stream) {
  using namespace mvb;
  int rc = kv4_check(cache);
  if (rc != kOk) return rc;
  if (num_tokens < 0 || num_q_heads < 0) return kInvalidArgument;
  const int d = cache->head_dim;
  if (cos_sin != nullptr) {
    if (!positions || max_pos <= 0 || rotary_dim <= 0) return kInvalidArgument;
    if (rotary_dim > d || rotary_dim % 16 != 0) return kUnsupportedShape;
  }
  if (num_tokens == 0) return kOk;
  if (k == v && k_in_place && cos_sin != nullptr) return kInvalidArgument;   // (values are read by other warps than those that turn the keys)
  if (!k || !v || !slot_mapping || (num_q_heads > 0 && (!q || !q_out))) return kInvalidArgument;
  if ((num_q_heads > 0 && (q_row_stride % 8 || q_out_row_stride % 8)) || k_row_stride % 8 || v_row_stride % 8) return kMisaligned;
  if (!is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(cos_sin, 16) || (num_q_heads > 0 && (!is_aligned(q, 16) || !is_aligned(q_out, 16))))
    return kMisaligned;
  Kv4WriteParams p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.k = static_cast<__nv_bfloat16*>(k); p.v = static_cast<const __nv_bfloat16*>(v);
  p.q_stride = q_row_stride; p.qo_stride = q_out_row_stride; p.k_stride = k_row_stride; p.v_stride = v_row_stride;
  p.positions = positions; p.cos_sin = cos_sin; p.max_pos = max_pos; p.slots = slot_mapping;
  p.k_codes = static_cast<uint8_t*>(cache->k_codes); p.v_codes = static_cast<uint8_t*>(cache->v_codes);
  p.k_affine = static_cast<uint32_t*>(cache->k_affine); p.v_affine = static_cast<uint32_t*>(cache->v_affine);
  p.num_slots = cache->num_blocks * cache->block_size;
  p.by_block = FastDiv(static_cast<uint32_t>(cache->block_size));
  p.tokens = num_tokens; p.hq = num_q_heads; p.hkv = cache->num_kv_heads; p.block_size = cache->block_size;
  p.rot = cos_sin != nullptr ? rotary_dim : 0; p.k_in_place = k_in_place; p.dev_status = dev_status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_head_dim(d, [&](auto tag) -> int {
    constexpr int D = decltype(tag)::value;
    constexpr int RPW = 32 / (D / 8);
    auto warps_of = [&](int heads, int items) -> int { return (heads + RPW * items - 1) / (RPW * items); };
    // four rows in flight per lane where that still leaves every SM 12 warps, one where there are few tokens (8 KV heads of 128, one and four
    // rows: 96 tokens 2.5 and 3.1 us; 512 tokens with 32 heads of queries 5.4 and 4.4, with 16 4.4 and 3.8; 16384 with 32 131 and 87)
    const int items = static_cast<int64_t>(num_tokens) * (warps_of(p.hq, 4) + 2 * warps_of(p.hkv, 4)) >= static_cast<int64_t>(sm_count()) * 12 ? 4 : 1;
    Kv4WriteParams r = p;
    r.q_warps = warps_of(p.hq, items); r.k_warps = warps_of(p.hkv, items);
    const int64_t per_token = r.q_warps + 2 * static_cast<int64_t>(r.k_warps), warps = per_token * num_tokens;
    if (warps > 0x7fffffffLL - 8) return kUnsupportedShape;
    r.by_token = FastDiv(static_cast<uint32_t>(per_token));
    const unsigned grid = static_cast<unsigned>((warps + 7) / 8);
    if (items == 4 && interleaved) kv4_write_kernel<D, true, 4><<<grid, 256, 0, st>>>(r);
    else if (items == 4) kv4_write_kernel<D, false, 4><<<grid, 256, 0, st>>>(r);
    else if (interleaved) kv4_write_kernel<D, true, 1><<<grid, 256, 0, st>>>(r);
    else kv4_write_kernel<D, false, 1><<<grid, 256, 0, st>>>(r);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
  });
}

extern "C" int mvb_kv4_gather(const mvb_kv4_cache* cache, const int32_t* cu_seqlens_k, const int32_t* block_table, int64_t table_stride,
                              int table_width, int num_seqs, int num_rows, void* k_out, void* v_out, int32_t* dev_status, void* stream) {
  using namespace mvb;
  int rc = kv4_check(cache);
  if (rc != kOk) return rc;
  if (num_seqs < 0 || num_rows < 0) return kInvalidArgument;
  if (num_seqs == 0 || num_rows == 0) return kOk;
  if (!cu_seqlens_k || !block_table || !k_out || !v_out || table_width <= 0 || table_stride < table_width) return kInvalidArgument;
  if (!is_aligned(k_out, 16) || !is_aligned(v_out, 16)) return kMisaligned;
  Kv4GatherParams p;
  p.k_codes = static_cast<const uint32_t*>(cache->k_codes); p.v_codes = static_cast<const uint32_t*>(cache->v_codes);
  p.k_affine = static_cast<const uint32_t*>(cache->k_affine); p.v_affine = static_cast<const uint32_t*>(cache->v_affine);
  p.k_out = static_cast<__nv_bfloat16*>(k_out); p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.cu = cu_seqlens_k; p.block_table = block_table; p.table_stride = table_stride; p.num_blocks = cache->num_blocks;
  p.by_block = FastDiv(static_cast<uint32_t>(cache->block_size));
  p.table_width = table_width; p.num_seqs = num_seqs; p.rows = num_rows; p.hkv = cache->num_kv_heads; p.block_size = cache->block_size;
  p.dev_status = dev_status;
  return by_head_dim(cache->head_dim, [&](auto tag) -> int {
    constexpr int D = decltype(tag)::value;
    constexpr int RPW = 32 / (D / 8), ITEMS = D == 256 ? 2 : 4;
    const int64_t groups = (static_cast<int64_t>(p.hkv) + RPW - 1) / RPW, per_token = (groups + ITEMS - 1) / ITEMS;
    const int64_t warps = per_token * num_rows;
    if (warps > 0x7fffffffLL - 8) return kUnsupportedShape;
    Kv4GatherParams r = p;
    r.by_token = FastDiv(static_cast<uint32_t>(per_token));
    kv4_gather_kernel<D, ITEMS><<<static_cast<unsigned>((warps + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(r);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
  });
}
