// Which spans of 64 cached tokens a query should read.
//
// Every span has, per KV head and channel, the least and the greatest key of its tokens (bf16 [blocks, kv heads, block_size / 64, 2, D]).
// For a query the sum over the channels of max(q least, q greatest) is a bound on q . k for every key of the span; the bounds of a group's
// query heads are added up, and the spans with the greatest sums are read, the first and the last one always.
//
// The sums decide which tokens are read, so they must not depend on the order of summation: a product of two bf16 is exact in fp32 and
// the sum runs in fp64, where 53 bits hold it exactly unless its products span more than 2^27.
#include "dtype.cuh"
#include "host_util.cuh"
#include "kv4.cuh"

#include <type_traits>

namespace mvb {

struct SummariseParams {
  const uint32_t *k_codes, *k_affine;
  const int32_t* slots;
  __nv_bfloat16* summaries;
  int64_t num_slots;
  int tokens, hkv, block_size;
  int* dev_status;
};

// A warp per (token, head): the last of a step's tokens inside a span renews the span's bounds from the rows up to its own.  A token is the
// last one when the next row of the step does not follow it in the same span.
template <int D>
__global__ void __launch_bounds__(256) kv4_summarise_kernel(const SummariseParams p) {
  constexpr int LPH = D / 8, RPW = 32 / LPH;
  constexpr uint32_t FULL = 0xffffffffu;
  const int lane = threadIdx.x & 31, c = lane % LPH, sub = lane / LPH;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const int64_t slot = p.slots[t];
  if (slot < 0 || slot >= p.num_slots) {
    if (slot != -1 && lane == 0 && blockIdx.y == 0) report(p.dev_status, kDevBadSlot, static_cast<int>(t));
    return;
  }
  const int end = static_cast<int>(slot % kKv4Span);
  if (end != kKv4Span - 1 && t + 1 < p.tokens && p.slots[t + 1] == slot + 1) return;
  const int h = blockIdx.y;
  const int64_t block = slot / p.block_size;
  const int in_block = static_cast<int>(slot - block * p.block_size), span = in_block / kKv4Span;
  const int64_t row0 = kv4_row(block, p.hkv, h, p.block_size, span * kKv4Span);
  float lo[8], hi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) { lo[e] = INFINITY; hi[e] = -INFINITY; }
#pragma unroll 4
  for (int r = sub; r <= end; r += RPW) {
    float y[8];
    kv4_values(__ldg(p.k_codes + (row0 + r) * (D / 8) + kv4_word<D>(c, true)), __ldg(p.k_affine + (row0 + r) * (D / 64) + (c >> 3)), y);
#pragma unroll
    for (int e = 0; e < 8; ++e) { lo[e] = fminf(lo[e], y[e]); hi[e] = fmaxf(hi[e], y[e]); }
  }
#pragma unroll
  for (int off = LPH; off < 32; off <<= 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = fminf(lo[e], __shfl_xor_sync(FULL, lo[e], off));
      hi[e] = fmaxf(hi[e], __shfl_xor_sync(FULL, hi[e], off));
    }
  }
  __nv_bfloat16* out = p.summaries + ((block * p.hkv + h) * (p.block_size / kKv4Span) + span) * (2 * D);
  if (sub == 0) {
    store_vec<__nv_bfloat16, 8>(out + c * 8, lo);
    store_vec<__nv_bfloat16, 8>(out + D + c * 8, hi);
  }
}

struct SelectParams {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const __nv_bfloat16* summaries;
  const int32_t* seqlens;
  const int32_t* block_table;
  int64_t table_stride, num_blocks;
  int32_t* out;
  int table_width, hkv, group, block_size, budget;
  int* dev_status;
};

constexpr int kSelectThreads = 256;
constexpr int kSelectMaxSpans = 16384;       // keys of 8 bytes in shared memory: a context of 1 M tokens
constexpr int kSelectMaxGroup = 8;

// ascending with the sum, whatever its sign
__device__ __forceinline__ uint64_t order_key(double x) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(x));
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

// exclusive sum over the block's threads; every thread also gets the total
__device__ __forceinline__ int block_prefix(int v, int* scratch, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    const int s = scratch[w];
    before += w < warp ? s : 0;
    total += s;
  }
  return before + x - v;
}

// A block per (KV head, sequence): the sums, then the budget-th greatest by radix selection on their bits, eight at a time, then the
// chosen indices in order (of equal sums the lower ones).
template <int D>
__global__ void __launch_bounds__(kSelectThreads) kv4_select_kernel(const SelectParams p) {
  constexpr uint32_t FULL = 0xffffffffu;
  constexpr int CPL = D / 32;                                // channels of a lane
  extern __shared__ uint64_t keys[];
  __shared__ int hist[256], scratch[kSelectThreads / 32], pick_s[2];
  const int h = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = p.seqlens[b];
  int32_t* out = p.out + (static_cast<int64_t>(b) * p.hkv + h) * p.budget;
  int count = n > 0 ? (n + kKv4Span - 1) / kKv4Span : 0;
  const int most = p.table_width * (p.block_size / kKv4Span);
  if (count > most) {                                        // a length that its block list does not hold
    if (threadIdx.x == 0) report(p.dev_status, kDevBadLength, b);
    count = most;
  }
  if (count <= p.budget) {
    for (int i = threadIdx.x; i < p.budget; i += kSelectThreads) out[i] = i < count ? i : -1;
    return;
  }
  float q[kSelectMaxGroup][CPL];
#pragma unroll
  for (int g = 0; g < kSelectMaxGroup; ++g) {
#pragma unroll
    for (int e = 0; e < CPL; ++e)
      q[g][e] = g < p.group ? __bfloat162float(p.q[b * p.q_stride + (static_cast<int64_t>(h) * p.group + g) * D + lane * CPL + e]) : 0.f;
  }
  const int per_block = p.block_size / kKv4Span;
  for (int s = warp; s < count; s += kSelectThreads / 32) {
    const int64_t block = p.block_table[b * p.table_stride + s / per_block];
    double sum = 0.0;
    if (block >= 0 && block < p.num_blocks) {
      const __nv_bfloat16* at = p.summaries + ((block * p.hkv + h) * per_block + s % per_block) * (2 * D) + lane * CPL;
      float lo[CPL], hi[CPL];
#pragma unroll
      for (int e = 0; e < CPL; e += 2) {
        const uint32_t a = __ldg(reinterpret_cast<const uint32_t*>(at + e)), z = __ldg(reinterpret_cast<const uint32_t*>(at + D + e));
        lo[e] = bf16_lo(a); lo[e + 1] = bf16_hi(a); hi[e] = bf16_lo(z); hi[e + 1] = bf16_hi(z);
      }
#pragma unroll
      for (int g = 0; g < kSelectMaxGroup; ++g) {
        if (g < p.group) {
#pragma unroll
          for (int e = 0; e < CPL; ++e) sum += static_cast<double>(fmaxf(q[g][e] * lo[e], q[g][e] * hi[e]));
        }
      }
    } else if (lane == 0) {
      report(p.dev_status, kDevBadBlock, b);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(FULL, sum, off);
    if (lane == 0) keys[s] = s == 0 || s == count - 1 ? ~0ull : order_key(sum);
  }
  __syncthreads();
  uint64_t prefix = 0, mask = 0;
  int need = p.budget;                                       // still to be found among the keys that share the prefix
  for (int shift = 56; shift >= 0; shift -= 8) {
    hist[threadIdx.x] = 0;
    __syncthreads();
    for (int s = threadIdx.x; s < count; s += kSelectThreads) {
      const uint64_t k = keys[s];
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    const int bin = 255 - static_cast<int>(threadIdx.x), mine = hist[bin];
    int total;
    const int above = block_prefix(mine, scratch, total);    // keys in greater bins
    if (above < need && above + mine >= need) { pick_s[0] = bin; pick_s[1] = need - above; }
    __syncthreads();
    prefix |= static_cast<uint64_t>(pick_s[0]) << shift;
    mask |= 255ull << shift;
    need = pick_s[1];
    const bool all = hist[pick_s[0]] == need;                // every key of this bin is taken
    __syncthreads();
    if (all) { need = 0x7fffffff; break; }
  }
  // a thread walks a run of neighbouring spans; keys equal to the prefix (under the mask) are taken up to `need`, the lower indices first
  const int run = (count + kSelectThreads - 1) / kSelectThreads;
  const int first = min(static_cast<int>(threadIdx.x) * run, count), last = min(first + run, count);
  int equal = 0, over = 0, total;
  for (int s = first; s < last; ++s) {
    const uint64_t k = keys[s] & mask;
    equal += k == prefix;
    over += k > prefix;
  }
  const int equal_before = block_prefix(equal, scratch, total);
  const int equal_taken = max(0, min(equal, need - equal_before));
  int at = block_prefix(over + equal_taken, scratch, total);
  int left = equal_taken;
  for (int s = first; s < last; ++s) {
    const uint64_t k = keys[s] & mask;
    if (k > prefix || (k == prefix && left > 0)) {
      left -= k == prefix;
      if (at < p.budget) out[at] = s;
      ++at;
    }
  }
}

}  // namespace mvb

extern "C" int mvb_kv4_summarise(const mvb_kv4_cache* cache, const int32_t* slot_mapping, int num_tokens, void* summaries,
                                 int32_t* dev_status, void* stream) {
  using namespace mvb;
  const int rc = kv4_check(cache);
  if (rc != kOk) return rc;
  if (num_tokens < 0) return kInvalidArgument;
  if (num_tokens == 0) return kOk;
  if (!slot_mapping || !summaries) return kInvalidArgument;
  if (!is_aligned(summaries, 16)) return kMisaligned;
  if (cache->num_kv_heads > 65535) return kUnsupportedShape;
  SummariseParams p;
  p.k_codes = static_cast<const uint32_t*>(cache->k_codes); p.k_affine = static_cast<const uint32_t*>(cache->k_affine);
  p.slots = slot_mapping; p.summaries = static_cast<__nv_bfloat16*>(summaries);
  p.num_slots = cache->num_blocks * cache->block_size;
  p.tokens = num_tokens; p.hkv = cache->num_kv_heads; p.block_size = cache->block_size; p.dev_status = dev_status;
  const dim3 grid((static_cast<unsigned>(num_tokens) + 7) / 8, cache->num_kv_heads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cache->head_dim == 64) kv4_summarise_kernel<64><<<grid, 256, 0, st>>>(p);
  else if (cache->head_dim == 128) kv4_summarise_kernel<128><<<grid, 256, 0, st>>>(p);
  else kv4_summarise_kernel<256><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
}

extern "C" int mvb_kv4_select(const void* q, int64_t q_row_stride, const void* summaries, int64_t num_blocks, int block_size,
                              const int32_t* cache_seqlens, const int32_t* block_table, int64_t table_stride, int table_width, int num_seqs,
                              int num_q_heads, int num_kv_heads, int head_dim, int budget, int32_t* spans, int32_t* dev_status, void* stream) {
  using namespace mvb;
  if (num_seqs < 0 || num_blocks <= 0 || block_size <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || table_width <= 0 || budget < 2)
    return kInvalidArgument;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return kUnsupportedShape;
  if (num_q_heads % num_kv_heads != 0 || num_q_heads / num_kv_heads > kSelectMaxGroup || block_size % kKv4Span != 0) return kUnsupportedShape;
  if (static_cast<int64_t>(table_width) * (block_size / kKv4Span) > kSelectMaxSpans || num_seqs > 65535) return kUnsupportedShape;
  if (num_seqs == 0) return kOk;
  if (!q || !summaries || !cache_seqlens || !block_table || !spans || table_stride < table_width) return kInvalidArgument;
  if (!is_aligned(q, 2) || !is_aligned(summaries, 16)) return kMisaligned;
  SelectParams p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.q_stride = q_row_stride; p.summaries = static_cast<const __nv_bfloat16*>(summaries);
  p.seqlens = cache_seqlens; p.block_table = block_table; p.table_stride = table_stride; p.num_blocks = num_blocks; p.out = spans;
  p.table_width = table_width; p.hkv = num_kv_heads; p.group = num_q_heads / num_kv_heads; p.block_size = block_size; p.budget = budget;
  p.dev_status = dev_status;
  const size_t smem = sizeof(uint64_t) * static_cast<size_t>(table_width) * (block_size / kKv4Span);
  const dim3 grid(num_kv_heads, num_seqs);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto tag) -> int {
    constexpr int D = decltype(tag)::value;
    struct Tag {};
    if (smem > 40 * 1024) {
      const int rc = opt_in_dynamic_smem<Tag>(reinterpret_cast<const void*>(&kv4_select_kernel<D>), smem);
      if (rc != kOk) return rc;
    }
    kv4_select_kernel<D><<<grid, kSelectThreads, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
  };
  if (head_dim == 64) return launch(std::integral_constant<int, 64>{});
  if (head_dim == 128) return launch(std::integral_constant<int, 128>{});
  return launch(std::integral_constant<int, 256>{});
}
