// Attention of one new token per sequence over the 4-bit cache.
//
//     out = sum_t softmax_t(f(q . k_t scale)) v_t        k_t = m + s c per group of 64 channels, v_t likewise; f the score cap, if any
//
// over all tokens of the sequence, the last `window_left` + 1 of them, or the tokens of a list of 64-token spans per sequence and KV head.
#include "dtype.cuh"
#include "host_util.cuh"
#include "kv4.cuh"

#include <type_traits>

namespace mvb {

struct Decode4Params {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  int64_t q_stride, out_stride;
  const uint32_t *k_codes, *v_codes, *k_affine, *v_affine;
  const int32_t* seqlens;
  const int32_t* block_table;
  const int32_t* spans;                // [num_seqs, hkv, budget] or nullptr
  int64_t table_stride, num_blocks;
  FastDiv by_block;
  int table_width, num_seqs, hkv, group, block_size, budget, window_left;
  float scale_log2, cap_in, cap_log2, out_scale;
  int* dev_status;
};

constexpr int kDecode4MaxGroup = 8;

// A block per (KV head, sequence); a warp walks every eighth token of it, a lane holds D / 32 channels.
template <int D, bool CAP>
__global__ void __launch_bounds__(256) kv4_decode_kernel(const Decode4Params p) {
  constexpr uint32_t FULL = 0xffffffffu;
  constexpr int W = D / 8, G = kDecode4MaxGroup, CPL = D / 32;
  extern __shared__ float sh[];                              // [8 warps][G][D + 2]
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = p.seqlens[b];
  float q[G][CPL], o[G][CPL], m[G], l[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = -INFINITY; l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < CPL; ++e) {
      q[g][e] = g < p.group ? __bfloat162float(p.q[b * p.q_stride + (static_cast<int64_t>(h) * p.group + g) * D + lane * CPL + e]) : 0.f;
      o[g][e] = 0.f;
    }
  }
  const int32_t* list = p.spans != nullptr ? p.spans + (static_cast<int64_t>(b) * p.hkv + h) * p.budget : nullptr;
  const int first = list == nullptr && p.window_left >= 0 ? max(0, n - 1 - p.window_left) : 0;
  const int steps = list != nullptr ? p.budget * kKv4Span : n;
  for (int i = first + warp; i < steps; i += 8) {
    int t = i;
    if (list != nullptr) {
      const int span = list[i / kKv4Span];
      if (span < 0 || span > (n - 1) / kKv4Span) continue;
      t = span * kKv4Span + i % kKv4Span;
      if (t >= n) continue;
    }
    const int col = p.by_block.div(t);
    const int64_t block = col < p.table_width ? p.block_table[b * p.table_stride + col] : -1;
    if (block < 0 || block >= p.num_blocks) {
      if (lane == 0) report(p.dev_status, kDevBadBlock, b);
      continue;
    }
    const int64_t row = kv4_row(block, p.hkv, h, p.block_size, t - col * p.block_size);
    float k[CPL], v[CPL];
    const int L = lane * CPL / 8, e0 = lane * CPL % 8;
    const uint32_t kw = p.k_codes[row * W + kv4_word<D>(L, true)], vw = p.v_codes[row * W + kv4_word<D>(L, false)];
    const uint32_t ka = p.k_affine[row * (D / 64) + L / 8], va = p.v_affine[row * (D / 64) + L / 8];
#pragma unroll
    for (int e = 0; e < CPL; ++e) {
      k[e] = fmaf(kv4_scale(ka), static_cast<float>((kw >> kv4_shift(e0 + e)) & 15u), kv4_min(ka));
      v[e] = fmaf(kv4_scale(va), static_cast<float>((vw >> kv4_shift(e0 + e)) & 15u), kv4_min(va));
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (g >= p.group) continue;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < CPL; ++e) s = fmaf(q[g][e], k[e], s);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(FULL, s, off);
      const float x = CAP ? p.cap_log2 * tanhf(s * p.cap_in) : s * p.scale_log2;
      const float nm = fmaxf(m[g], x), a = exp2f(m[g] - nm), w = exp2f(x - nm);
      m[g] = nm;
      l[g] = l[g] * a + w;
#pragma unroll
      for (int e = 0; e < CPL; ++e) o[g][e] = o[g][e] * a + w * v[e];
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float* at = sh + (warp * G + g) * (D + 2);
#pragma unroll
    for (int e = 0; e < CPL; ++e) at[lane * CPL + e] = o[g][e];
    if (lane == 0) { at[D] = m[g]; at[D + 1] = l[g]; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.group * D; i += 256) {
    const int g = i / D, e = i % D;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int w = 0; w < 8; ++w) M = fmaxf(M, sh[(w * G + g) * (D + 2) + D]);
    for (int w = 0; w < 8; ++w) {
      const float* at = sh + (w * G + g) * (D + 2);
      const float f = at[D] == -INFINITY ? 0.f : exp2f(at[D] - M);
      L += f * at[D + 1]; O += f * at[e];
    }
    p.out[b * p.out_stride + (static_cast<int64_t>(h) * p.group + g) * D + e] = __float2bfloat16_rn(L > 0.f ? O / L * p.out_scale : 0.f);
  }
}

}  // namespace mvb

extern "C" size_t mvb_decode_attn4_workspace_bytes(int max_seqs, int num_q_heads, int num_kv_heads, int head_dim) {
  if (max_seqs <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
  return 256;
}

extern "C" int mvb_decode_attn4(const void* q, int64_t q_row_stride, const mvb_kv4_cache* cache, const int32_t* cache_seqlens,
                                const int32_t* block_table, int64_t table_stride, int table_width, const int32_t* spans, int budget,
                                int num_seqs, int num_q_heads, float scale, int window_left, float softcap, float out_scale, void* out,
                                int64_t out_row_stride, void* workspace, size_t workspace_bytes, int32_t* dev_status, void* stream) {
  using namespace mvb;
  const int rc = kv4_check(cache);
  if (rc != kOk) return rc;
  if (num_seqs < 0 || num_q_heads <= 0 || table_width <= 0 || table_stride < table_width || !(softcap >= 0.f)) return kInvalidArgument;
  if (spans != nullptr && (budget <= 0 || window_left >= 0)) return kInvalidArgument;
  if (num_q_heads % cache->num_kv_heads != 0 || num_q_heads / cache->num_kv_heads > kDecode4MaxGroup) return kUnsupportedShape;
  if (num_seqs == 0) return kOk;
  if (!q || !out || !cache_seqlens || !block_table || !workspace) return kInvalidArgument;
  if (q_row_stride % 8 || out_row_stride % 8 || !is_aligned(q, 16) || !is_aligned(out, 16) || !is_aligned(workspace, 256)) return kMisaligned;
  if (num_seqs > 65535) return kUnsupportedShape;
  (void)workspace_bytes;
  const float kLog2e = 1.4426950408889634f;
  Decode4Params p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.q_stride = q_row_stride; p.out = static_cast<__nv_bfloat16*>(out); p.out_stride = out_row_stride;
  p.k_codes = static_cast<const uint32_t*>(cache->k_codes); p.v_codes = static_cast<const uint32_t*>(cache->v_codes);
  p.k_affine = static_cast<const uint32_t*>(cache->k_affine); p.v_affine = static_cast<const uint32_t*>(cache->v_affine);
  p.seqlens = cache_seqlens; p.block_table = block_table; p.table_stride = table_stride; p.table_width = table_width; p.spans = spans;
  p.num_blocks = cache->num_blocks; p.by_block = FastDiv(static_cast<uint32_t>(cache->block_size));
  p.num_seqs = num_seqs; p.hkv = cache->num_kv_heads; p.group = num_q_heads / cache->num_kv_heads; p.block_size = cache->block_size;
  p.budget = budget; p.window_left = window_left;
  p.scale_log2 = scale * kLog2e; p.cap_in = softcap > 0.f ? scale / softcap : 0.f; p.cap_log2 = softcap * kLog2e; p.out_scale = out_scale;
  p.dev_status = dev_status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto tag, auto cap) -> int {
    constexpr int D = decltype(tag)::value;
    struct Tag {};
    const size_t smem = sizeof(float) * 8 * kDecode4MaxGroup * (D + 2);
    const int r = opt_in_dynamic_smem<Tag>(reinterpret_cast<const void*>(&kv4_decode_kernel<D, decltype(cap)::value>), smem);
    if (r != kOk) return r;
    kv4_decode_kernel<D, decltype(cap)::value><<<dim3(p.hkv, num_seqs), 256, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
  };
  auto by_cap = [&](auto tag) -> int { return softcap > 0.f ? launch(tag, std::true_type{}) : launch(tag, std::false_type{}); };
  if (cache->head_dim == 64) return by_cap(std::integral_constant<int, 64>{});
  if (cache->head_dim == 128) return by_cap(std::integral_constant<int, 128>{});
  return by_cap(std::integral_constant<int, 256>{});
}
