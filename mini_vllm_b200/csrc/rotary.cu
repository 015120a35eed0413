// Rotation of queries and keys by position (an elementwise pass, bound by memory): neighbouring pairs (2i, 2i + 1) or halves
// (i, i + R/2) of the first R channels of a head, the others carried along.
//     y_a = x_a cos - x_b sin,   y_b = x_b cos + x_a sin        with cos, sin of (position, i) from the caller's fp32 table
// Products and sum are rounded one by one in fp32, then once to the activation type, as the write kernels of the other caches do.
//
// 16384 tokens of 32 + 8 heads of 128, half of each turned: 0.34 GB in 53 us, 6.4 TB/s (0.98 of what a copy reaches).
//
// A unit is one 16-byte vector of a head with its partner (halves), or by itself (neighbours and the channels carried along); shapes or
// addresses that do not allow vectors take units of one pair.  In place, the channels behind R are not touched.
#include "dtype.cuh"
#include "host_util.cuh"
#include "kv4.cuh"

#include <type_traits>

namespace mvb {

struct RotaryParams {
  const void *q, *k;
  void *q_out, *k_out;
  int64_t q_stride, k_stride, qo_stride, ko_stride;
  const int64_t* positions;
  const float* cos_sin;
  int64_t max_pos;
  int tokens, hq, hkv, d, rot;
  int rot_units, units;                // of one head
  int64_t total;
  FastDiv by_token, by_head;
  int* dev_status;
};

template <int V>
__device__ __forceinline__ void load_table(const float* p, float (&out)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 w = __ldg(reinterpret_cast<const float4*>(p + i));
      out[i] = w.x; out[i + 1] = w.y; out[i + 2] = w.z; out[i + 3] = w.w;
    }
  } else if constexpr (V == 2) {
    const float2 w = __ldg(reinterpret_cast<const float2*>(p));
    out[0] = w.x; out[1] = w.y;
  } else {
    out[0] = __ldg(p);
  }
}

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = a;
  a = __fsub_rn(__fmul_rn(x, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(x, s));
}

// V elements to a vector (1: a unit is one pair of elements).  A thread takes the same unit of HEADS neighbouring heads of a token, so that
// it loads the unit's angles once, and requests all of them before it turns the first.
template <class T, int V, bool INTER, int HEADS>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  constexpr bool PAIR = !(INTER && V > 1);                   // a unit's partners are two vectors
  constexpr int N = PAIR ? V : V / 2;                        // angles of a unit
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.total) return;
  const int half = p.rot / 2, heads = p.hq + p.hkv;
  const uint32_t t = p.by_token.div(static_cast<uint32_t>(i));
  const uint32_t in_token = static_cast<uint32_t>(i) - t * p.by_token.n;
  const uint32_t group = p.by_head.div(in_token);
  const int unit = static_cast<int>(in_token - group * p.by_head.n), head0 = static_cast<int>(group) * HEADS;
  const bool turned = unit < p.rot_units;
  const int one = !turned ? p.rot + (unit - p.rot_units) * V : PAIR && INTER ? 2 * unit : unit * V;
  const int two = INTER ? one + 1 : one + half;
  const int64_t pos = turned ? __ldg(p.positions + t) : 0;
  auto at = [&](int head, bool out) -> T* {
    const bool is_q = head < p.hq;
    const T* base = static_cast<const T*>(out ? (is_q ? p.q_out : p.k_out) : (is_q ? p.q : p.k));
    const int64_t stride = out ? (is_q ? p.qo_stride : p.ko_stride) : (is_q ? p.q_stride : p.k_stride);
    return const_cast<T*>(base) + static_cast<int64_t>(t) * stride + static_cast<int64_t>(is_q ? head : head - p.hq) * p.d;
  };
  using Raw = std::conditional_t<V == 1, T, uint4>;          // as it lies in memory, until its turn
  Raw a[HEADS], b[HEADS];
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    if (head0 + j < heads) {
      const T* src = at(head0 + j, false);
      a[j] = *reinterpret_cast<const Raw*>(src + one);
      if (PAIR && turned) b[j] = *reinterpret_cast<const Raw*>(src + two);
    }
  }
  const bool ok = pos >= 0 && pos < p.max_pos;
  float c[N], s[N];
  if (turned) {
    if (!ok) report(p.dev_status, kDevBadPosition, static_cast<int>(t));
    const float* row = p.cos_sin + (ok ? pos : 0) * p.rot + unit * N;
    load_table<N>(row, c);
    load_table<N>(row + half, s);
  }
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    if (head0 + j >= heads) break;
    T* dst = at(head0 + j, true);
    if (turned) {
      float x[V], y[V];
      load_vec<T, V>(reinterpret_cast<const T*>(&a[j]), x);
      if constexpr (PAIR) load_vec<T, V>(reinterpret_cast<const T*>(&b[j]), y);
      if (ok) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if constexpr (PAIR) turn(x[e], y[e], c[e], s[e]);
          else turn(x[2 * e], x[2 * e + 1], c[e], s[e]);
        }
      }
      store_vec<T, V>(dst + one, x);
      if constexpr (PAIR) store_vec<T, V>(dst + two, y);
    } else {
      *reinterpret_cast<Raw*>(dst + one) = a[j];
    }
  }
}

template <class T>
static int launch_rotary(RotaryParams& p, bool inter, cudaStream_t stream) {
  constexpr int V = kVec<T>;
  const bool in_place = p.q == p.q_out && p.k == p.k_out;
  const bool vec = p.d % V == 0 && p.rot % (inter ? V : 2 * V) == 0 && p.q_stride % V == 0 && p.k_stride % V == 0 && p.qo_stride % V == 0 &&
                   p.ko_stride % V == 0 && is_aligned(p.q, 16) && is_aligned(p.k, 16) && is_aligned(p.q_out, 16) && is_aligned(p.k_out, 16) &&
                   is_aligned(p.cos_sin, 16);
  const int v = vec ? V : 1;
  p.rot_units = vec && inter ? p.rot / V : p.rot / 2 / v;
  p.units = p.rot_units + (in_place ? 0 : (p.d - p.rot) / v);
  const int heads = p.hq + p.hkv;
  // four heads a thread where that still leaves every SM 512 threads, one where there are few tokens (32 + 8 heads of 128, whole heads turned
  // by neighbours, one and four heads: 96 tokens 2.0 and 2.4 us, 512 3.6 and 3.4, 1024 5.7 and 4.9, 16384 73 and 55; by halves 2.1 and 2.8, 3.2
  // and 3.4, 5.1 and 4.8, 66 and 58)
  const bool many = vec && static_cast<int64_t>((heads + 3) / 4) * p.units * p.tokens >= static_cast<int64_t>(sm_count()) * 512;
  const int64_t per_token = static_cast<int64_t>(many ? (heads + 3) / 4 : heads) * p.units;
  if (per_token > 0x7fffffffLL / (p.tokens > 0 ? p.tokens : 1)) return kUnsupportedShape;
  p.total = per_token * p.tokens;
  p.by_token = FastDiv(static_cast<uint32_t>(per_token));
  p.by_head = FastDiv(static_cast<uint32_t>(p.units));
  const unsigned grid = static_cast<unsigned>((p.total + 255) / 256);
  if (many && inter) rotary_kernel<T, V, true, 4><<<grid, 256, 0, stream>>>(p);
  else if (many) rotary_kernel<T, V, false, 4><<<grid, 256, 0, stream>>>(p);
  else if (vec && inter) rotary_kernel<T, V, true, 1><<<grid, 256, 0, stream>>>(p);
  else if (vec) rotary_kernel<T, V, false, 1><<<grid, 256, 0, stream>>>(p);
  else if (inter) rotary_kernel<T, 1, true, 1><<<grid, 256, 0, stream>>>(p);
  else rotary_kernel<T, 1, false, 1><<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
}

}  // namespace mvb

extern "C" int mvb_rotary(const void* q, int64_t q_row_stride, const void* k, int64_t k_row_stride, void* q_out, int64_t q_out_row_stride,
                          void* k_out, int64_t k_out_row_stride, const int64_t* positions, const float* cos_sin, int64_t max_pos,
                          int num_tokens, int num_q_heads, int num_kv_heads, int head_dim, int rotary_dim, int interleaved, int dtype,
                          int32_t* dev_status, void* stream) {
  using namespace mvb;
  if (num_tokens < 0 || num_q_heads < 0 || num_kv_heads < 0 || head_dim <= 0 || rotary_dim <= 0 || max_pos <= 0) return kInvalidArgument;
  if (num_q_heads == 0 && num_kv_heads == 0) return kInvalidArgument;
  if (rotary_dim % 2 != 0 || rotary_dim > head_dim || (dtype != kBf16 && dtype != kF32)) return kUnsupportedShape;
  if (num_tokens == 0) return kOk;
  if ((num_q_heads > 0 && (!q || !q_out)) || (num_kv_heads > 0 && (!k || !k_out)) || !positions || !cos_sin) return kInvalidArgument;
  const uintptr_t size = dtype == kBf16 ? 2 : 4;
  if (!is_aligned(q, size) || !is_aligned(k, size) || !is_aligned(q_out, size) || !is_aligned(k_out, size) || !is_aligned(positions, 8) ||
      !is_aligned(cos_sin, 4))
    return kMisaligned;
  RotaryParams p;
  p.q = num_q_heads > 0 ? q : nullptr; p.k = num_kv_heads > 0 ? k : nullptr;
  p.q_out = num_q_heads > 0 ? q_out : nullptr; p.k_out = num_kv_heads > 0 ? k_out : nullptr;
  p.q_stride = num_q_heads > 0 ? q_row_stride : 0; p.k_stride = num_kv_heads > 0 ? k_row_stride : 0;
  p.qo_stride = num_q_heads > 0 ? q_out_row_stride : 0; p.ko_stride = num_kv_heads > 0 ? k_out_row_stride : 0;
  p.positions = positions; p.cos_sin = cos_sin; p.max_pos = max_pos;
  p.tokens = num_tokens; p.hq = num_q_heads; p.hkv = num_kv_heads; p.d = head_dim; p.rot = rotary_dim;
  p.dev_status = dev_status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == kBf16 ? launch_rotary<__nv_bfloat16>(p, interleaved != 0, st) : launch_rotary<float>(p, interleaved != 0, st);
}
