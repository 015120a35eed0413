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

// of two numbers; of anything and what is not one, that
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

struct SummariseParams {
  const uint32_t *k_codes, *k_affine;
  const int32_t* slots;
  __nv_bfloat16* summaries;
  int64_t num_slots;
  int tokens, hkv, block_size;
  int* dev_status;
};

// The last of a step's tokens inside a span renews the span's bounds from the rows up to its own; a token is the last one when the next row
// of the step does not follow it in the same span.  WARPS warps share a (token, head): eight where a step has few tokens (decoding: nearly
// every token is such a last one, and a span is then one round of loads), one where it has many (prompts: one token in 64 has work).
template <int D, int WARPS>
__global__ void __launch_bounds__(256) kv4_summarise_kernel(const SummariseParams p) {
  constexpr int LPH = D / 8, RPW = 32 / LPH, ROUNDS = kKv4Span / (RPW * WARPS);
  constexpr uint32_t FULL = 0xffffffffu;
  __shared__ float part_s[WARPS > 1 ? WARPS : 1][2][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane % LPH, sub = lane / LPH;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (8 / WARPS) + (WARPS > 1 ? 0 : warp);
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
  const int first = (WARPS > 1 ? warp : 0) * RPW + sub;
  float lo[8], hi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) { lo[e] = INFINITY; hi[e] = -INFINITY; }
  constexpr int AT_ONCE = ROUNDS < 8 ? ROUNDS : 8;
#pragma unroll 1
  for (int base = 0; base < ROUNDS; base += AT_ONCE) {
    uint32_t word[AT_ONCE], affine[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int r = first + (base + i) * RPW * WARPS;
      if (r <= end) {
        word[i] = __ldg(p.k_codes + (row0 + r) * (D / 8) + kv4_word<D>(c, true));
        affine[i] = __ldg(p.k_affine + (row0 + r) * (D / 64) + (c >> 3));
      }
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      if (first + (base + i) * RPW * WARPS <= end) {
        float y[8];
        kv4_values(word[i], affine[i], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) { lo[e] = min_nan(lo[e], y[e]); hi[e] = max_nan(hi[e], y[e]); }
      }
    }
  }
#pragma unroll
  for (int off = LPH; off < 32; off <<= 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = min_nan(lo[e], __shfl_xor_sync(FULL, lo[e], off));
      hi[e] = max_nan(hi[e], __shfl_xor_sync(FULL, hi[e], off));
    }
  }
  __nv_bfloat16* out = p.summaries + ((block * p.hkv + h) * (p.block_size / kKv4Span) + span) * (2 * D);
  if constexpr (WARPS == 1) {
    if (sub == 0) {
      store_vec<__nv_bfloat16, 8>(out + c * 8, lo);
      store_vec<__nv_bfloat16, 8>(out + D + c * 8, hi);
    }
  } else {
    if (sub == 0) {
      store_f32<8>(&part_s[warp][0][c * 8], lo);
      store_f32<8>(&part_s[warp][1][c * 8], hi);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += 256) {
      const int side = i / D, e = i % D;
      float y = part_s[0][side][e];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) y = side ? max_nan(y, part_s[w][side][e]) : min_nan(y, part_s[w][side][e]);
      out[i] = __float2bfloat16_rn(y);
    }
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
  int max_spans, hkv, group, block_size, budget;
  int* dev_status;
};

constexpr int kSelectThreads = 256;
constexpr int kSelectMaxSpans = 16384;       // keys of 8 bytes in shared memory: a context of 1 M tokens
constexpr int kSelectMaxGroup = 8;

// ascending with the sum, whatever its sign; a sum that is not a number comes before all others, so that what made it is read
__device__ __forceinline__ uint64_t order_key(double x) {
  if (x != x) return ~0ull;
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

// A cluster of CL blocks per (KV head, sequence).  Its blocks share the spans and send their sums' bits, as keys that ascend with the sum, to the
// first one, which finds the budget-th greatest by radix selection, eight bits at a time from the first one in which keys differ, and
// writes the chosen indices in order (of equal sums the lower ones).  Eight lanes take a span, so that a warp has four spans in flight.
// Bound by latency: for few rows by the chain of loads, sums and ranking (4 sequences of 9000-40000 tokens, 8 KV heads: 11 us, 67 with one block
// and one span a warp), for many by the same chain in every block, loads and barriers at 45 % of the issue slots (96 sequences: 26 us).
template <int D>
__global__ void __launch_bounds__(kSelectThreads) kv4_select_kernel(const SelectParams p) {
  constexpr uint32_t FULL = 0xffffffffu;
  constexpr int PIECES = D / 64;                             // of eight channels, of a lane
  extern __shared__ uint64_t keys[];
  __shared__ __align__(16) float q_s[kSelectMaxGroup * D];
  __shared__ int hist[256], scratch[kSelectThreads / 32], pick_s[2];
  __shared__ unsigned long long differ_s;
  uint32_t cl, rank;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cl));
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int h = blockIdx.x / cl, b = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & 7;
  const int n = p.seqlens[b];
  int32_t* out = p.out + (static_cast<int64_t>(b) * p.hkv + h) * p.budget;
  int count = n > 0 ? (n - 1) / kKv4Span + 1 : 0;
  const int per_block = p.block_size / kKv4Span;
  if (count > p.max_spans) {                                 // longer than the caller said, or than its block list holds
    if (threadIdx.x == 0) report(p.dev_status, kDevBadLength, b);
    count = p.max_spans;
  }
  if (count <= p.budget) {                                   // (the whole cluster)
    if (rank == 0)
      for (int i = threadIdx.x; i < p.budget; i += kSelectThreads) out[i] = i < count ? i : -1;
    return;
  }
  if (cl > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // (every block has begun before one writes to another)
  const int32_t* table = p.block_table + b * p.table_stride;
  for (int i = threadIdx.x; i < p.group * D; i += kSelectThreads)
    q_s[i] = __bfloat162float(p.q[b * p.q_stride + static_cast<int64_t>(h) * p.group * D + i]);
  if (threadIdx.x == 0) differ_s = 0;
  __syncthreads();
  if (cl > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  uint32_t keys_0;                                           // the first block's keys, in the cluster's shared memory
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(keys_0) : "r"(smem_u32(keys)));
  constexpr int NS = D == 256 ? 1 : 2;                       // spans that eight lanes have in flight
  const int stride = cl * (kSelectThreads / 8) * NS;
  for (int base = (rank * (kSelectThreads / 32) + warp) * 4 * NS; base < count; base += stride) {     // warp-uniform
    uint4 lo[NS][PIECES], hi[NS][PIECES];
    bool ok[NS];
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int s = base + 4 * k + (lane >> 3);
      const bool inner = s > 0 && s < count - 1;             // the first and the last one are taken anyway
      int64_t block = -1;
      if (inner) block = __ldg(table + s / per_block);
      ok[k] = block >= 0 && block < p.num_blocks;
      if (inner && !ok[k] && sub == 0) report(p.dev_status, kDevBadBlock, b);
      const uint4* at = reinterpret_cast<const uint4*>(p.summaries + ((ok[k] ? block * p.hkv + h : 0) * per_block + (ok[k] ? s % per_block : 0)) * (2 * D));
#pragma unroll
      for (int i = 0; i < PIECES; ++i) { lo[k][i] = __ldg(at + i * 8 + sub); hi[k][i] = __ldg(at + D / 8 + i * 8 + sub); }
    }
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int s = base + 4 * k + (lane >> 3);
      double sum = 0.0, sum2 = 0.0;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const uint32_t l[4] = {lo[k][i].x, lo[k][i].y, lo[k][i].z, lo[k][i].w}, u[4] = {hi[k][i].x, hi[k][i].y, hi[k][i].z, hi[k][i].w};
        for (int g = 0; g < p.group; ++g) {
          float q[8];
          load_f32<8>(q_s + g * D + (i * 8 + sub) * 8, q);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sum += static_cast<double>(fmaxf(q[2 * e] * bf16_lo(l[e]), q[2 * e] * bf16_lo(u[e])));
            sum2 += static_cast<double>(fmaxf(q[2 * e + 1] * bf16_hi(l[e]), q[2 * e + 1] * bf16_hi(u[e])));
          }
        }
      }
      sum += sum2;
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) sum += __shfl_xor_sync(FULL, sum, off);
      if (sub == 0 && s < count) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(keys_0 + 8u * s), "l"(order_key(ok[k] ? sum : 0.0)));
    }
  }
  if (cl > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  // ---- the first block: which of the inner spans -------------------------------------------------------------------------------------
  // Up to 256 spans a thread has one and counts the better ones: no passes, one prefix sum.  That takes every warp the whole list, so blocks
  // that share an SM with others do it up to 128 (8 pairs of 250 spans: 8.6 us against 10.1 by radix; 768 pairs of 90 spans 23.3 and 24.5, of
  // 250 54.9 and 51.0)
  if (count <= (cl > 1 ? kSelectThreads : kSelectThreads / 2)) {
    const int s = threadIdx.x;
    const bool ends = s == 0 || s == count - 1;
    int better = s < count ? 0 : count;
    if (warp * 32 < count) {
      const uint64_t own = s < count ? keys[s] : 0;
      // spans before the warp's own count from equality on, those behind it above, and inside it depends on the lane
      const int first = max(1, warp * 32), last = min(count - 1, warp * 32 + 32);
#pragma unroll 8
      for (int o = 1; o < first; ++o) better += keys[o] >= own;
#pragma unroll 4
      for (int o = first; o < last; ++o) {
        const uint64_t k = keys[o];
        better += k > own || (k == own && o < s);
      }
#pragma unroll 8
      for (int o = last; o < count - 1; ++o) better += keys[o] > own;
    }
    const bool take = ends || better < p.budget - 2;
    int total;
    const int at = block_prefix(take ? 1 : 0, scratch, total);
    if (take && at < p.budget) out[at] = s;
    return;
  }
  const uint64_t sample = keys[1];
  uint64_t differ = 0;
  for (int s = 1 + threadIdx.x; s < count - 1; s += kSelectThreads) differ |= keys[s] ^ sample;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) differ |= __shfl_xor_sync(FULL, differ, off);
  if (lane == 0 && differ != 0) atomicOr(&differ_s, static_cast<unsigned long long>(differ));
  __syncthreads();
  differ = differ_s;
  int top = 64 - __clzll(static_cast<long long>(differ));    // bits from here on are the same in all keys
  uint64_t mask = top == 64 ? 0 : ~0ull << top, prefix = sample & mask;
  int need = p.budget - 2;                                   // still to be found among the keys that share the prefix
  while (top > 0 && need > 0) {
    const int shift = max(top - 8, 0), width = top - shift;
    hist[threadIdx.x] = 0;
    __syncthreads();
    for (int s = 1 + threadIdx.x; s < count - 1; s += kSelectThreads) {
      const uint64_t k = keys[s];
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << width) - 1)], 1);
    }
    __syncthreads();
    const int bin = 255 - static_cast<int>(threadIdx.x), mine = hist[bin];
    int total;
    const int above = block_prefix(mine, scratch, total);    // keys in greater bins
    if (above < need && above + mine >= need) { pick_s[0] = bin; pick_s[1] = need - above; }
    __syncthreads();
    prefix |= static_cast<uint64_t>(pick_s[0]) << shift;
    mask |= ((1ull << width) - 1) << shift;
    need = pick_s[1];
    top = shift;
    const bool all = hist[pick_s[0]] == need;                // every key that shares the prefix is taken
    __syncthreads();
    if (all) break;
  }
  // a thread walks a run of neighbouring spans; keys equal to the prefix (under the mask) are taken up to `need`, the lower indices first
  const int run = (count + kSelectThreads - 1) / kSelectThreads;
  const int first = min(static_cast<int>(threadIdx.x) * run, count), last = min(first + run, count);
  int equal = 0, over = 0, total;
  for (int s = first; s < last; ++s) {
    const uint64_t k = keys[s] & mask;
    const bool ends = s == 0 || s == count - 1;
    over += ends || k > prefix;
    equal += !ends && k == prefix;
  }
  const int equal_before = block_prefix(equal, scratch, total);
  int left = max(0, min(equal, need - equal_before));
  int at = block_prefix(over + left, scratch, total);
  for (int s = first; s < last; ++s) {
    const uint64_t k = keys[s] & mask;
    const bool ends = s == 0 || s == count - 1;
    bool take = ends || k > prefix;
    if (!take && k == prefix && left > 0) { take = true; --left; }
    if (take) {
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // a block for each (token, head) of a step of few, a warp for each of many (decoding, 8 heads of 128, eight warps and one: 32 sequences 2.9
  // and 5.1 us, 128 5.5 and 5.3, 1024 27 and 18; prompts: 64 tokens 2.5 and 4.5, 512 4.6 and 4.5, 8192 39 and 15)
  const bool few = static_cast<int64_t>(num_tokens) * cache->num_kv_heads <= 1024;
  const dim3 grid(few ? num_tokens : (static_cast<unsigned>(num_tokens) + 7) / 8, cache->num_kv_heads);
  auto launch = [&](auto tag) -> int {
    constexpr int D = decltype(tag)::value;
    if (few) kv4_summarise_kernel<D, 8><<<grid, 256, 0, st>>>(p);
    else kv4_summarise_kernel<D, 1><<<grid, 256, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
  };
  if (cache->head_dim == 64) return launch(std::integral_constant<int, 64>{});
  if (cache->head_dim == 128) return launch(std::integral_constant<int, 128>{});
  return launch(std::integral_constant<int, 256>{});
}

extern "C" int mvb_kv4_select(const void* q, int64_t q_row_stride, const void* summaries, int64_t num_blocks, int block_size,
                              const int32_t* cache_seqlens, const int32_t* block_table, int64_t table_stride, int table_width, int num_seqs,
                              int num_q_heads, int num_kv_heads, int head_dim, int max_tokens, int budget, int32_t* spans,
                              int32_t* dev_status, void* stream) {
  using namespace mvb;
  if (num_seqs < 0 || num_blocks <= 0 || block_size <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || table_width <= 0 || max_tokens <= 0 || budget < 2)
    return kInvalidArgument;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return kUnsupportedShape;
  if (num_q_heads % num_kv_heads != 0 || num_q_heads / num_kv_heads > kSelectMaxGroup || block_size % kKv4Span != 0) return kUnsupportedShape;
  if (num_seqs > 65535) return kUnsupportedShape;
  // keys in shared memory: for the longest context that may come
  int64_t spans_most = static_cast<int64_t>(table_width) * (block_size / kKv4Span);
  const int64_t said = (static_cast<int64_t>(max_tokens) + kKv4Span - 1) / kKv4Span;
  if (said < spans_most) spans_most = said;
  if (spans_most > kSelectMaxSpans) return kUnsupportedShape;
  if (num_seqs == 0) return kOk;
  if (!q || !summaries || !cache_seqlens || !block_table || !spans || table_stride < table_width) return kInvalidArgument;
  if (!is_aligned(q, 2) || !is_aligned(summaries, 16)) return kMisaligned;
  SelectParams p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.q_stride = q_row_stride; p.summaries = static_cast<const __nv_bfloat16*>(summaries);
  p.seqlens = cache_seqlens; p.block_table = block_table; p.table_stride = table_stride; p.num_blocks = num_blocks; p.out = spans;
  p.max_spans = static_cast<int>(spans_most); p.hkv = num_kv_heads; p.group = num_q_heads / num_kv_heads; p.block_size = block_size; p.budget = budget;
  p.dev_status = dev_status;
  const size_t smem = sizeof(uint64_t) * static_cast<size_t>(spans_most);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // a cluster of at most eight blocks for one (sequence, head): up to 5/3 blocks per SM, and 44 spans of the longest context for each.  128-wide
  // heads, clusters of 1, 2, 4, 8: 32 pairs of 16 K tokens 16.7, 11.5, 8.6, 10.6 us, of 40 K 34.6, 22.2, 16.4, 14.8; 72 of 40 K 35.1, 22.5, 21.4,
  // 22.7; 128 of 16 K 17.0, 14.6, 16.6, 25.2; 256 of 16 K 22.0, 26.4, 27.6, 43.4
  const int64_t pairs = static_cast<int64_t>(num_kv_heads) * num_seqs;
  int cl = 1;
  while (cl < 8 && pairs * cl * 3 < 5 * sm_count() && spans_most >= 88 * cl) cl *= 2;
  auto launch = [&](auto tag) -> int {
    constexpr int D = decltype(tag)::value;
    struct Tag {};
    if (smem > 32 * 1024) {
      const int rc = opt_in_dynamic_smem<Tag>(reinterpret_cast<const void*>(&kv4_select_kernel<D>), smem);
      if (rc != kOk) return rc;
    }
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cl; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(num_kv_heads) * cl, num_seqs);
    cfg.blockDim = dim3(kSelectThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_select_kernel<D>, p) == cudaSuccess ? kOk : kLaunchFailed;
  };
  if (head_dim == 64) return launch(std::integral_constant<int, 64>{});
  if (head_dim == 128) return launch(std::integral_constant<int, 128>{});
  return launch(std::integral_constant<int, 256>{});
}
