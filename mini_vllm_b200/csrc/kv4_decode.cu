// Attention of one new token per sequence over the 4-bit cache.
//
//     out = sum_t softmax_t(f(q . k_t scale)) v_t        k_t = m + s c per group of 64 channels, v_t likewise; f the score cap, if any
//
// over all tokens of the sequence, the last `window_left` + 1 of them, or the tokens of a list of 64-token spans per sequence and KV head.
//
// Nothing is unpacked to values.  With the codes themselves as matrix operands (masked halves of a word are fp16 subnormals, kv4.cuh)
//     q . k_t  = sum over groups of  s_t (q . c_t) + m_t sum(q)
//     sum_t p_t v_t = sum over t of  (p_t s_t) c_t  +  sum_t p_t m_t        per group
// so a 32-bit word of eight codes costs five integer instructions, for keys (one shift, four ANDs) and for values (where two tokens of a
// channel have to meet in a register: a byte permutation, and the high codes of a byte are never masked out, their sums are those of
// whole bytes less those of the low codes), and scales and minima cost a few per token.  q is brought to [2^14, 2^15)
// by a power of two per head so that fp16 holds every bf16 exactly down to 2^-29 of the greatest; the channels whose codes sit at bits 4-7
// (16 times as large) have it divided by 16.  Scores, softmax statistics and outputs are fp32; the weights p s are rounded once, to fp16.  Every
// group of channels and head has a power of two of its own on them, moved when the group's greatest weight would pass 2^14: they never
// overflow, and a group keeps its bits whatever the sizes of other groups, tokens and heads (scales from 2^-120 on; p itself is at most 2^-14, so
// that a warp's sum of p m is finite too, for 16 K tokens of the largest values there are).  A rounding of p s meets the codes, up to 15 of them,
// while p m is exact: next to the plain form's error that is 2^-11 sum p (15 s) more at most.
//
// On paper bound by memory: a tile of 32 tokens of a 128-wide head is 4608 bytes.  Its 650 warp instructions, most of them on the integer
// pipe, bring instruction issue near: 240 sequences of 128-8192 tokens, 16 heads on 8, 0.51 GB in 115 us, 4.4 TB/s (0.68 of what a copy reaches),
// 62 % of the issue slots, the integer pipe at 59 %.  Neither is at its limit: four warps a scheduler, at 128 registers with 156 bytes of them
// spilled, do not cover each other's waits, and more do not fit.  A few rows are bound by the chain of dependent loads (lengths, block lists,
// tiles, parts): one context of 700 tokens 10 us.
//
// Work is tiles of 32 tokens of one (sequence, head), numbered sequence by sequence and head by head.  Each CTA takes a contiguous range (all
// alike, or, where there are few rows, a share of one of them), each of its warps a contiguous part of that.  A warp streams its tiles
// through a private ring in shared memory (cp.async, 16 bytes a lane, placed so that the fragment loads meet no bank twice) and needs no
// other warp until its range is done.  Rows that lie within one warp's range go straight to the output; parts of a row are put together by
// the CTA, and where a row crosses CTAs by the warps that arrive last.  Every warp works the split out for itself from the lengths, so
// there is no plan to make, the grid does not depend on data, and nothing ever waits for another CTA.
#include "dtype.cuh"
#include "host_util.cuh"
#include "kv4.cuh"

#include <type_traits>

namespace mvb {

constexpr int kDecode4MaxGroup = 8;
constexpr int kDecode4MaxCtas = 160;

constexpr int kDecode4MaxWarps = 16;

template <int D, int W>
struct Decode4Cfg {
  static constexpr int TOK = 32;                             // tokens of a tile
  static constexpr int NW = W;                               // warps of a CTA
  static constexpr int NST = 2;                              // tiles in a warp's ring, one of them being computed (three: 113 us instead of 111 for the ragged batch, when that took 111)
  static constexpr int CODES = TOK * D / 2, AFF = TOK * D / 16;
  static constexpr int STAGE = 2 * CODES + 2 * AFF;          // key codes, value codes, key affine, value affine
  static constexpr int RING = NST * STAGE;
  static constexpr int GRP = D / 64;                         // groups of channels
  static constexpr int WK = D / 32, WV = D / 64;             // 32-bit words of a lane: of a key, of a value
  static constexpr int PART = 8 * D * 4;                     // a part of a row: outputs of up to eight heads
  static constexpr size_t SMEM = static_cast<size_t>(NW) * (RING + PART);
  static_assert(PART <= RING, "a warp's last part takes the place of its ring");
};

// floats of a part that a CTA leaves for others: outputs of the group's heads, then their log2-sum-exps, one copy for each warp that merges
// a share of the channels
__host__ __device__ __forceinline__ constexpr int decode4_part(int group, int d) {
  return group * d + kDecode4MaxGroup * kDecode4MaxWarps;
}

struct Decode4Params {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  int64_t q_stride, out_stride;
  const uint8_t *k_codes, *v_codes, *k_affine, *v_affine;
  const int32_t* seqlens;
  const int32_t* block_table;
  const int32_t* spans;                // [num_seqs, hkv, budget] or nullptr
  int64_t table_stride, num_blocks;
  FastDiv by_block;
  int table_width, max_len, num_seqs, hkv, group, block_size, budget, window_left;
  float scale_log2, cap_in, cap_log2, out_scale;
  float* parts;                        // [CTAs][2]: of the CTA's first row and of its last
  int32_t* arrivals;                   // [num_seqs * hkv][warps], zero between launches
  int* dev_status;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(                                                       // (not volatile: the compiler may interleave the products of a tile)
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Powers of two, as their exponents say: of a whole number (0 below 2^-126, at most 2^127, and that of what is no number: nothing has been added up
// then), one over 2^-126 .. 2^126, and what brings the greatest of a group's weights to 2^8 .. 2^9
constexpr float kMostUp = 0x1p126f;
__device__ __forceinline__ float pow2_whole(float x) {
  return __uint_as_float(static_cast<uint32_t>(static_cast<int>(fmaxf(fminf(x, 127.f), -127.f)) + 127) << 23);
}
__device__ __forceinline__ float pow2_inverse(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }
__device__ __forceinline__ float up_for(float most) {
  const int e = static_cast<int>(__float_as_uint(most) >> 23) - 127;
  return __uint_as_float(static_cast<uint32_t>(127 + max(min(8 - e, 126), -102)) << 23);
}
// the outputs of a group's channels, by a factor for each of the two heads
template <int N>
__device__ __forceinline__ void scale_group(float (&o)[N][4], int j, float a, float b) {
#pragma unroll
  for (int i = 4 * j; i < 4 * j + 4; ++i) { o[i][0] *= a; o[i][1] *= b; o[i][2] *= a; o[i][3] *= b; }
}
template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* at, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(at);
  } else if constexpr (N == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(at);
    w[0] = u.x; w[1] = u.y;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(at);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  }
}

// Where things lie in a stage.  The rows that the lanes of a fragment read together are 0, 3, 4, 7 or 1, 2, 5, 6 of eight (values) and
// pairs of one even and one odd row (keys), see decode4_row; 16-byte pieces change places with the row so that these meet in no bank.
template <int D>
__device__ __forceinline__ uint32_t key_piece(int t, int piece) {           // byte of a row's 16-byte piece
  return t * (D / 2) + ((D == 256 ? piece ^ (t & 1) : piece) << 4);
}
template <int D>
__device__ __forceinline__ uint32_t value_piece(int t, int piece) {
  if (D == 256) return t * 128 + ((piece ^ (t & 6)) << 4);
  if (D == 128) return t * 64 + ((piece ^ ((t >> 1) & 2)) << 4);
  return (t ^ ((t >> 1) & 2)) * 32 + (piece << 4);
}
// the token (of eight) that stands in row r of a fragment
__device__ __forceinline__ int decode4_row(int r) { return r ^ ((r >> 1) & 1); }

// The tiles of a (sequence, head) row, one after the other.  Tile 0 holds no tokens: it stands for what a row costs besides them (its q, its
// end; 1.7 us against 2.0 for a tile, with all SMs busy), so that warps with many short rows get no more work than the others.
template <int TOK>
struct Decode4Walk {
  int b, h, i, count, n;               // tile i of `count` of head h of sequence b, which has n tokens
  __device__ __forceinline__ static int length(const Decode4Params& p, int b) {
    return min(p.seqlens[b], p.max_len);
  }
  __device__ __forceinline__ static int first_tile(const Decode4Params& p, int n) {
    return p.window_left >= 0 ? max(0, n - 1 - p.window_left) / TOK : 0;
  }
  __device__ __forceinline__ static int tiles(const Decode4Params& p, int n) {
    if (n <= 0) return 0;
    if (p.spans != nullptr) return 1 + (kKv4Span / TOK) * min(p.budget, (n + kKv4Span - 1) / kKv4Span);
    return 1 + (n + TOK - 1) / TOK - first_tile(p, n);
  }
  __device__ __forceinline__ void next(const Decode4Params& p) {
    if (++i < count) return;
    i = 0;
    if (++h < p.hkv) return;
    h = 0;
    do {
      if (++b >= p.num_seqs) { count = 0x7fffffff; n = 0; return; }         // past the last row: nobody reads on
      n = length(p, b);
      count = tiles(p, n);
    } while (count == 0);
  }
};

// How `total` tiles are dealt to the CTAs: no more of these than give every warp a tile (rows of a small call stay on few of them), the
// first `rest` of them one tile more than the others.
struct Decode4Cut {
  int ctas, per, rest;
  __device__ __forceinline__ Decode4Cut(int total, int warps) {
    ctas = min(static_cast<int>(gridDim.x), (total + warps - 1) / warps);
    per = ctas > 0 ? total / ctas : 0;
    rest = total - per * ctas;
  }
  __device__ __forceinline__ int start(int c) const { return c * per + min(c, rest); }
  __device__ __forceinline__ int of(int tile) const { return tile < rest * (per + 1) ? tile / (per + 1) : (tile - rest) / per; }
};

// a run of tiles of head h of sequence b (n tokens): its first token (behind the span's, with a list of spans) and which lane has its block (none: -1)
struct Decode4Run {
  int known, known_row, sel, token, tiles, b, h, n;
};

// a CTA's tiles and, where whole CTAs are given to rows, the first CTA of its row and their number (first < 0: the even cut)
struct Decode4Share {
  int t0, t1, first, parts;
};

template <int D, bool CAP, int W>
__global__ void __launch_bounds__(W * 32, 1) kv4_decode_kernel(const Decode4Params p) {
  using C = Decode4Cfg<D, W>;
  using Walk = Decode4Walk<C::TOK>;
  constexpr int NW = C::NW, NT = NW * 32, NST = C::NST, GRP = C::GRP;
  constexpr uint32_t FULL = 0xffffffffu, LO = 0x000f000fu, HI = 0x00f000f0u, BYTE = 0x00ff00ffu;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int total_s;
  __shared__ Decode4Share cut_s;
  __shared__ int meta_s[NW][2][3];                           // a warp's parts: row (-1: none), the row's first tile and the one behind its last
  __shared__ Walk fs_s[NW], cs_s[NW];                        // a warp's fetching and computing side
  __shared__ Decode4Run run_s[NW];
  __shared__ int before_s[NW];                               // entries that name a span in front of the known ones
  __shared__ __align__(16) float lse_s[2][kDecode4MaxGroup][NW];            // log2-sum-exps of the warps' first and last parts, -inf: none

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c4 = lane & 3;
  const int G = p.group;

  // ---- the split.  Every warp works it out for itself: lane i sums up the tiles of the i-th run of neighbouring sequences ---------------
  const int cta = blockIdx.x;
  const int lane_seqs = (p.num_seqs + 31) / 32, b0 = min(lane * lane_seqs, p.num_seqs), b1 = min(b0 + lane_seqs, p.num_seqs);
  auto tiles_of = [&](int b) -> int { return Walk::tiles(p, Walk::length(p, b)); };
  auto before_me = [&](int own, int& sum) -> int {           // exclusive sum over the lanes, and all of them
    int x = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(FULL, x, off);
      if (lane >= off) x += y;
    }
    sum = __shfl_sync(FULL, x, 31);
    return x - own;
  };
  int own = 0, some = 0, total;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    const int n = p.seqlens[b];
    if (n > p.max_len && warp == 0) report(p.dev_status, kDevBadLength, b);
    const int v = Walk::tiles(p, min(n, p.max_len));
    own += v;
    some += v > 0;
  }
  const int pre = before_me(own, total);
  some = __reduce_add_sync(FULL, some);
  total *= p.hkv;
  if (some < p.num_seqs) {                                   // sequences without a token: zeros
    for (int b = cta; b < p.num_seqs; b += gridDim.x) {
      if (p.seqlens[b] <= 0) {
        for (int e = threadIdx.x; e < p.hkv * G * D / 8; e += NT)
          *reinterpret_cast<uint4*>(p.out + b * p.out_stride + e * 8) = make_uint4(0, 0, 0, 0);
      }
    }
  }
  // Few rows: whole CTAs for each of them, in proportion to its tiles but one for a row of up to three tiles a warp, so that a CTA works on one
  // row and most need no other CTA.  Where some CTA would get much more than its share, or there are more rows than CTAs: the even cut.
  // (Cut evenly and by rows: 8 rows of 22 tiles 12.7 and 10.3 us, with sixteen warps 17.9 and 13.2; 128 rows of up to 17 tiles of 256-wide heads
  // 17.3 and 14.4; 8 rows of 1280 25.3 and 22.1, with sixteen warps 30.2 and 26.6.)
  const int grid = gridDim.x, share = (total + grid - 1) / grid;
  const float part_of_grid = static_cast<float>(grid) / static_cast<float>(max(total, 1));
  auto ctas_of = [&](int v) -> int {                         // (a tile a warp at least: no CTA is left without one)
    return v == 0 ? 0 : v <= 3 * NW ? 1 : max(1, min(static_cast<int>(static_cast<float>(v) * part_of_grid), v / NW));
  };
  Decode4Share mine{0, 0, -1, 0};
  bool by_rows = false;
  if (static_cast<int64_t>(some) * p.hkv <= grid) {
    int ctas = 0, all;
    bool much = false;
    const int bound = share + share / 8 + 3 * NW;
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
      const int v = tiles_of(b), n = ctas_of(v);
      ctas += n * p.hkv;
      much |= v > n * bound;
    }
    const int pre_ctas = before_me(ctas, all);
    by_rows = !__any_sync(FULL, much) && all <= grid;
    if (by_rows) {
      if (cta >= all) return;
      int c = pre_ctas, at = pre, n = 1, v = 0;
      const bool here = cta >= pre_ctas && cta < pre_ctas + ctas;
      if (here) {
#pragma unroll 1
        for (int b = b0; b < b1; ++b, c += n * p.hkv, at += v) {
          v = tiles_of(b);
          n = ctas_of(v);
          if (cta < c + n * p.hkv) break;
        }
      }
      const int src = __ffs(__ballot_sync(FULL, here)) - 1;
      c = __shfl_sync(FULL, c, src); at = __shfl_sync(FULL, at, src); n = __shfl_sync(FULL, n, src); v = __shfl_sync(FULL, v, src);
      const int h = (cta - c) / n, i = cta - c - h * n, per = v / n, rest = v - per * n, t0 = (at * p.hkv + h * v) + i * per + min(i, rest);
      mine = Decode4Share{t0, t0 + per + (i < rest ? 1 : 0), cta - i, n};
    }
  }
  if (!by_rows) {
    const Decode4Cut cut(total, NW);
    if (cta >= cut.ctas) return;
    mine.t0 = cut.start(cta);
    mine.t1 = cut.start(cta + 1);
  }
  if (threadIdx.x == 0) { cut_s = mine; total_s = total; }
  int w0, w1;
  {
    const int tiles = mine.t1 - mine.t0;
    w0 = mine.t0 + warp * (tiles / NW) + min(warp, tiles % NW);
    w1 = w0 + tiles / NW + (warp < tiles % NW ? 1 : 0);
  }
  Walk cs;
  int row_t0 = 0;                                            // the number of the row's first tile
  {
    const int src = 31 - __clz(__ballot_sync(FULL, pre * p.hkv <= w0));     // whose sequences hold tile w0 (of a warp without tiles: anyone's)
    int b = b0, at = pre, v = 0;
    if (lane == src) {
#pragma unroll 1
      for (; b < b1; ++b, at += v) {
        v = tiles_of(b);
        if (w0 < (at + v) * p.hkv) break;
      }
    }
    cs.b = min(__shfl_sync(FULL, b, src), p.num_seqs - 1);
    at = __shfl_sync(FULL, at, src);
    cs.count = __shfl_sync(FULL, v, src);
    cs.n = Walk::length(p, cs.b);
    const int in_seq = w0 - at * p.hkv;
    cs.h = cs.count > 0 ? in_seq / cs.count : 0;
    cs.i = in_seq - cs.h * cs.count;
    row_t0 = w0 - cs.i;
  }
  if (lane < 2) meta_s[warp][lane][0] = -1;
  if (lane < kDecode4MaxGroup) lse_s[1][lane][warp] = -INFINITY;

  // ---- the fetching side ------------------------------------------------------------------------------------------------------------
  const uint32_t ring = smem_u32(smem) + warp * C::RING;
  int ft = w0;                                               // the next tile to fetch
  // A run: tiles that lie one behind the other in memory (of one block, or of one span).  Where the runs lie is known 32 at a time: lane i
  // has the block of table column known + i or, with a list of spans, the first token and the block of its entry known + i (no token: the
  // entry names no span of the sequence).  The i-th span of a row is the list's i-th entry that names one, wherever it stands.
  // What only changes from run to run is kept in shared memory.
  int u_block = -1, u_token = -1;
  if (lane == 0) { fs_s[warp] = cs; run_s[warp].known = 0; run_s[warp].known_row = -1; }
  __syncwarp();
  auto look = [&]() {                                        // the next run; its block may still be on its way
    if (ft >= w1) return;
    Walk fs = fs_s[warp];                                    // the first tile that no run covers yet
    if (fs.i == 0) {
      fs.i = 1;
      if (++ft >= w1) return;
    }
    int known = run_s[warp].known, known_row = run_s[warp].known_row, run_token;
    const int32_t* table = p.block_table + fs.b * p.table_stride;
    int at, room;
    if (p.spans == nullptr) {
      run_token = (Walk::first_tile(p, fs.n) + fs.i - 1) * C::TOK;
      at = static_cast<int>(p.by_block.div(run_token));
      room = ((at + 1) * p.block_size - run_token) / C::TOK;
      if (known_row != fs.b || at < known || at >= known + 32) {
        known = at; known_row = fs.b;
        u_block = at + lane < p.table_width ? __ldg(table + at + lane) : -1;
      }
    } else {
      constexpr int PER = kKv4Span / C::TOK;
      const int row = fs.b * p.hkv + fs.h, nth = (fs.i - 1) / PER;
      room = PER - (fs.i - 1) % PER;
      run_token = ((fs.i - 1) % PER) * C::TOK;
      int before = before_s[warp];
      if (known_row != row) { known = -32; before = 0; u_token = -1; known_row = row; }
      uint32_t named = __ballot_sync(FULL, u_token >= 0);
      bool more = false;
      while (nth >= before + __popc(named) && known + 32 < p.budget) {
        before += __popc(named);
        known += 32;
        const int span = known + lane < p.budget ? __ldg(p.spans + static_cast<int64_t>(row) * p.budget + known + lane) : -1;
        const bool fits = span <= (fs.n - 1) / kKv4Span;
        if (!fits) report(p.dev_status, kDevBadLength, fs.b);
        u_token = span >= 0 && fits ? span * kKv4Span : -1;
        named = __ballot_sync(FULL, u_token >= 0);
        more = true;
      }
      if (more) {
        u_block = u_token >= 0 ? __ldg(table + p.by_block.div(u_token)) : -1;
        if (lane == 0) before_s[warp] = before;
      }
      at = known + __ffs(__ballot_sync(FULL, u_token >= 0 && __popc(named & ((1u << lane) - 1)) == nth - before)) - 1;    // (known - 1: there is none)
    }
    const int tiles = min(room, fs.count - fs.i), b = fs.b, h = fs.h, n = fs.n;
    fs.i += tiles - 1;
    fs.next(p);
    __syncwarp();
    if (lane == 0) { fs_s[warp] = fs; run_s[warp] = Decode4Run{known, known_row, at - known, run_token, tiles, b, h, n}; }
    __syncwarp();
  };
  int f_stage = 0, f_left = 0, f_token = 0, f_n = 0;
  int64_t f_off = -1;                                        // of the codes, in bytes; < 0: nothing to read
  auto fetch = [&]() -> int {                                // the tile's first token, -1: nothing to read
    int first = -1;
    if (ft < w1) {
      if (f_left == 0) {                                     // on to the run that look() found
        const Decode4Run run = run_s[warp];
        const int block = __shfl_sync(FULL, u_block, run.sel & 31);
        f_token = run.token; f_left = run.tiles; f_n = run.n;
        bool ok = true;
        if (p.spans != nullptr) {
          const int base = __shfl_sync(FULL, u_token, run.sel & 31);
          ok = run.sel >= 0 && base >= 0;
          f_token = ok ? f_token + base : 0;
        }
        if (ok && (block < 0 || block >= p.num_blocks)) {
          if (lane == 0) report(p.dev_status, kDevBadBlock, run.b);
          ok = false;
        }
        const int in_block = f_token - static_cast<int>(p.by_block.div(max(f_token, 0))) * p.block_size;
        f_off = ok ? kv4_row(block, p.hkv, run.h, p.block_size, in_block) * (D / 2) : -1;
      }
      const bool ok = f_off >= 0 && f_token < f_n;
      first = ok ? f_token : -1;
      if (ok) {
        const uint8_t* k = p.k_codes + f_off + lane * 16;
        const uint8_t* v = p.v_codes + f_off + lane * 16;
        const uint32_t dst = ring + f_stage * C::STAGE;
        constexpr int PPR = D / 32;                          // 16-byte pieces of a row
#pragma unroll
        for (int i = 0; i < C::TOK * PPR / 32; ++i) {
          const int at = i * 32 + lane, t = at / PPR, piece = at % PPR;
          cp_async16(dst + key_piece<D>(t, piece), k + i * 512);
          cp_async16(dst + C::CODES + value_piece<D>(t, piece), v + i * 512);
        }
        const uint8_t* ka = p.k_affine + f_off / 8 + lane * 16;
        const uint8_t* va = p.v_affine + f_off / 8 + lane * 16;
        if constexpr (C::AFF / 16 >= 32) {
          cp_async16(dst + 2 * C::CODES + lane * 16, ka);
          cp_async16(dst + 2 * C::CODES + C::AFF + lane * 16, va);
        } else {
          constexpr int PA = C::AFF / 16;
          if (lane < 2 * PA) cp_async16(dst + 2 * C::CODES + lane * 16, lane < PA ? ka : va - PA * 16);
        }
        f_off += C::TOK * D / 2;
      }
      ++ft;
      f_token += C::TOK;
      f_stage = f_stage + 1 == NST ? 0 : f_stage + 1;
      if (--f_left == 0) look();
    }
    cp_async_commit();
    return first;
  };
  // q of a row, requested before anything that waits: word j of a lane is channels 8 (4 j + c4) .. of head g of the group
  uint4 qw[C::WK];
  auto ask_q = [&](int b, int h) {
#pragma unroll
    for (int j = 0; j < C::WK; ++j) {
      qw[j] = make_uint4(0, 0, 0, 0);
      if (g < G) qw[j] = __ldg(reinterpret_cast<const uint4*>(p.q + b * p.q_stride + (static_cast<int64_t>(h) * G + g) * D + 8 * (4 * j + c4)));
    }
  };
  if (w0 < w1) ask_q(cs.b, cs.h);
  if (lane == 0) cs_s[warp] = cs;
  look();
  static_assert(NST == 2, "one tile is on its way while another is computed");
  int on_its_way = fetch();

  // ---- the computing side -----------------------------------------------------------------------------------------------------------
  const int kt = decode4_row(g);                             // this lane's token of eight, in the roles of a key's row and of a score's
  const int vt0 = decode4_row(2 * c4), vt1 = decode4_row(2 * c4 + 1);
  int t = w0, stage = 0;
  while (t < w1) {
    const int n = cs_s[warp].n, row_t1 = row_t0 + cs_s[warp].count, seg_end = min(w1, row_t1);
    const int start = p.window_left >= 0 ? max(0, n - 1 - p.window_left) : 0;

    // q as the B operand (head g of the group in column g)
    uint32_t qf[C::WK][4];
    float qs_a[GRP], qs_b[GRP], f_a, f_b;                    // sums per group and the score's factor, of heads 2 c4 and 2 c4 + 1
    {
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < C::WK; ++j) {
        const uint32_t a[4] = {qw[j].x, qw[j].y, qw[j].z, qw[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) most = fmaxf(most, fmaxf(fabsf(bf16_lo(a[e])), fabsf(bf16_hi(a[e]))));
      }
      most = fmaxf(most, __shfl_xor_sync(FULL, most, 1));
      most = fmaxf(most, __shfl_xor_sync(FULL, most, 2));
      const int ex = static_cast<int>(__float_as_uint(most) >> 23) - 127;
      const int up = min(14 - ex, 126);
      const float grow = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
      float sum[GRP];
#pragma unroll
      for (int j = 0; j < GRP; ++j) sum[j] = 0.f;
#pragma unroll
      for (int j = 0; j < C::WK; ++j) {
        const uint32_t a[4] = {qw[j].x, qw[j].y, qw[j].z, qw[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = bf16_lo(a[e]) * grow, y = bf16_hi(a[e]) * grow;
          sum[j / 2] += x + y;
          const float less = (e & 1) ? 0.0625f : 1.f;        // their codes sit at bits 4-7
          qf[j][e] = pack_f16(x * less, y * less);
        }
      }
      // (a factor that fp32 holds: from 2^118 on, scores come out smaller than they are)
      const float f = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(min(127 + 24 - up, 254)) << 23);
#pragma unroll
      for (int j = 0; j < GRP; ++j) {
        sum[j] += __shfl_xor_sync(FULL, sum[j], 1);
        sum[j] += __shfl_xor_sync(FULL, sum[j], 2);
        sum[j] *= 0x1p-24f;
        qs_a[j] = __shfl_sync(FULL, sum[j], 8 * c4);
        qs_b[j] = __shfl_sync(FULL, sum[j], 8 * c4 + 4);
      }
      f_a = __shfl_sync(FULL, f, 8 * c4);
      f_b = __shfl_sync(FULL, f, 8 * c4 + 4);
    }
    float o[4 * C::WV][4], l_a = 0.f, l_b = 0.f, m_a = -INFINITY, m_b = -INFINITY, pm_a[GRP], pm_b[GRP];
    float2 up[GRP];                                          // what the group's weights are multiplied by, of the two heads
#pragma unroll
    for (int i = 0; i < 4 * C::WV; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int j = 0; j < GRP; ++j) { pm_a[j] = pm_b[j] = 0.f; up[j] = make_float2(kMostUp, kMostUp); }

    for (; t < seg_end; ++t) {
      if (t == row_t0) continue;                             // (the tile without tokens)
      cp_async_wait<NST - 2>();
      __syncwarp();                                          // the tile is there for every lane, and the one before has been read by all
      const int token0 = on_its_way;
      on_its_way = fetch();
      const uint8_t* at = smem + warp * C::RING + stage * C::STAGE;
      stage = stage + 1 == NST ? 0 : stage + 1;
      if (token0 < 0) continue;

      // ---- scores: rows are tokens, columns heads -------------------------------------------------------------------------------
      float x[2][4];
      uint32_t va[2][2][GRP];                                // (scale, minimum) of this lane's tokens: [16 tokens][upper eight][group]
      const bool whole = token0 >= start && token0 + C::TOK <= n;
      float ta = -INFINITY, tb = -INFINITY;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float acc[GRP][4];
#pragma unroll
        for (int j = 0; j < GRP; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
        uint32_t k0[C::WK], k1[C::WK];
        const int r0 = 16 * s + kt, r1 = r0 + 8;
        if constexpr (D == 64) {
          lds_words<2>(at + r0 * 32 + c4 * 8, k0);
          lds_words<2>(at + r1 * 32 + c4 * 8, k1);
        } else {
#pragma unroll
          for (int i = 0; i < C::WK / 4; ++i) {
            uint32_t u[4];
            lds_words<4>(at + key_piece<D>(r0, c4 * (C::WK / 4) + i), u);
#pragma unroll
            for (int e = 0; e < 4; ++e) k0[4 * i + e] = u[e];
            lds_words<4>(at + key_piece<D>(r1, c4 * (C::WK / 4) + i), u);
#pragma unroll
            for (int e = 0; e < 4; ++e) k1[4 * i + e] = u[e];
          }
        }
        uint32_t ka0[GRP], ka1[GRP];
        lds_words<GRP>(at + 2 * C::CODES + r0 * (D / 16), ka0);
        lds_words<GRP>(at + 2 * C::CODES + r1 * (D / 16), ka1);
        lds_words<GRP>(at + 2 * C::CODES + C::AFF + r0 * (D / 16), va[s][0]);
        lds_words<GRP>(at + 2 * C::CODES + C::AFF + r1 * (D / 16), va[s][1]);
#pragma unroll
        for (int j = 0; j < C::WK; ++j) {
          const uint32_t u = k0[j], w = k1[j], u8 = u >> 8, w8 = w >> 8;
          mma_f16_16816(acc[j / 2], u & LO, w & LO, u & HI, w & HI, qf[j][0], qf[j][1]);
          mma_f16_16816(acc[j / 2], u8 & LO, w8 & LO, u8 & HI, w8 & HI, qf[j][2], qf[j][3]);
        }
        x[s][0] = x[s][1] = x[s][2] = x[s][3] = 0.f;
#pragma unroll
        for (int j = 0; j < GRP; ++j) {
          const float s0 = kv4_scale(ka0[j]), s1 = kv4_scale(ka1[j]), m0 = kv4_min(ka0[j]), m1 = kv4_min(ka1[j]);
          x[s][0] = fmaf(s0, acc[j][0], fmaf(m0, qs_a[j], x[s][0]));
          x[s][1] = fmaf(s0, acc[j][1], fmaf(m0, qs_b[j], x[s][1]));
          x[s][2] = fmaf(s1, acc[j][2], fmaf(m1, qs_a[j], x[s][2]));
          x[s][3] = fmaf(s1, acc[j][3], fmaf(m1, qs_b[j], x[s][3]));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[s][i] *= (i & 1) ? f_b : f_a;                    // (rounded here: the weights' differences have to be those of one set of scores)
          if constexpr (CAP) x[s][i] = fmaf(-2.f * p.cap_log2, fast_rcp(1.f + fast_exp2(x[s][i] * p.cap_in)), p.cap_log2);
        }
        if (!whole) {                                        // tokens out of sight: no weight, whatever their rows hold
          const int j0 = token0 + r0, j1 = token0 + r1;
          if (j0 < start || j0 >= n) {
            x[s][0] = x[s][1] = -INFINITY;
#pragma unroll
            for (int j = 0; j < GRP; ++j) va[s][0][j] = 0u;
          }
          if (j1 < start || j1 >= n) {
            x[s][2] = x[s][3] = -INFINITY;
#pragma unroll
            for (int j = 0; j < GRP; ++j) va[s][1][j] = 0u;
          }
        }
        ta = fmax3(ta, x[s][0], x[s][2]);
        tb = fmax3(tb, x[s][1], x[s][3]);
      }
      // ---- the running reference, a whole number at least 14 above every score: weights stay below 2^-14, and old ones change by powers of two.
      // What the groups' weights are multiplied by moves against it, so that what has been added up stays as it is ----------------------------
      if (__any_sync(FULL, ta > m_a - 14.f || tb > m_b - 14.f)) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          ta = fmaxf(ta, __shfl_xor_sync(FULL, ta, off));
          tb = fmaxf(tb, __shfl_xor_sync(FULL, tb, off));
        }
        ta = fmaxf(m_a, ceilf(ta) + 20.f); tb = fmaxf(m_b, ceilf(tb) + 20.f);
        const float less_a = pow2_whole(m_a - ta), less_b = pow2_whole(m_b - tb), more_a = pow2_whole(ta - m_a), more_b = pow2_whole(tb - m_b);
        m_a = ta; m_b = tb;
        l_a *= less_a; l_b *= less_b;
#pragma unroll
        for (int j = 0; j < GRP; ++j) {
          pm_a[j] *= less_a; pm_b[j] *= less_b;
          const float2 to = make_float2(fminf(up[j].x * more_a, kMostUp), fminf(up[j].y * more_b, kMostUp));
          scale_group(o, j, to.x * pow2_inverse(up[j].x) * less_a, to.y * pow2_inverse(up[j].y) * less_b);
          up[j] = to;
        }
      }
      const float ra = m_a == -INFINITY ? 0.f : m_a, rb = m_b == -INFINITY ? 0.f : m_b;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        x[s][0] = fast_exp2(x[s][0] - ra); x[s][1] = fast_exp2(x[s][1] - rb); x[s][2] = fast_exp2(x[s][2] - ra); x[s][3] = fast_exp2(x[s][3] - rb);
        l_a += x[s][0] + x[s][2]; l_b += x[s][1] + x[s][3];
      }
      // ---- weights p s to fp16, each group's in a range of its own: its greatest is brought to 2^8 .. 2^9 when it would pass 2^14 ----------
      uint32_t w[2][GRP][2];
#pragma unroll 1
      for (bool again = true;;) {
        float most = 0.f;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int j = 0; j < GRP; ++j) {
            const float s0 = kv4_scale(va[s][0][j]), s1 = kv4_scale(va[s][1][j]);
            const float2 w0 = mul_f32x2(mul_f32x2(make_float2(x[s][0], x[s][1]), up[j]), make_float2(s0, s0));
            const float2 w1 = mul_f32x2(mul_f32x2(make_float2(x[s][2], x[s][3]), up[j]), make_float2(s1, s1));
            most = fmax3(fmax3(most, w0.x, w0.y), w1.x, w1.y);
            w[s][j][0] = pack_f16(w0.x, w0.y); w[s][j][1] = pack_f16(w1.x, w1.y);
          }
        }
        if (!__any_sync(FULL, most > 0x1p14f) || !again) break;             // (a weight that is not finite stays so)
        again = false;
#pragma unroll
        for (int j = 0; j < GRP; ++j) {
          float a = 0.f, b = 0.f;                            // the tile's greatest p s, of both heads
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const float s0 = kv4_scale(va[s][0][j]), s1 = kv4_scale(va[s][1][j]);
            a = fmax3(a, x[s][0] * s0, x[s][2] * s1);
            b = fmax3(b, x[s][1] * s0, x[s][3] * s1);
          }
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            a = fmaxf(a, __shfl_xor_sync(FULL, a, off));
            b = fmaxf(b, __shfl_xor_sync(FULL, b, off));
          }
          const float2 to = make_float2(fminf(up[j].x, up_for(a)), fminf(up[j].y, up_for(b)));
          scale_group(o, j, to.x * pow2_inverse(up[j].x), to.y * pow2_inverse(up[j].y));
          up[j] = to;
        }
      }
      // ---- transposed, as the B operand of the values -----------------------------------------------------------------------------------
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint32_t v00[C::WV], v01[C::WV], v10[C::WV], v11[C::WV];
        const int u0 = 16 * s + vt0, u1 = 16 * s + vt1;
        const uint8_t* vat = at + C::CODES;
        auto value = [&](int tok, uint32_t (&w)[C::WV]) {
          if constexpr (D == 256) lds_words<4>(vat + value_piece<D>(tok, g), w);
          else lds_words<C::WV>(vat + value_piece<D>(tok, D == 128 ? g >> 1 : g >> 2) + (D == 128 ? (g & 1) * 8 : (g & 3) * 4), w);
        };
        value(u0, v00); value(u1, v01); value(u0 + 8, v10); value(u1 + 8, v11);
#pragma unroll
        for (int j = 0; j < GRP; ++j) {
          const float m0 = kv4_min(va[s][0][j]), m1 = kv4_min(va[s][1][j]);
          pm_a[j] = fmaf(x[s][0], m0, fmaf(x[s][2], m1, pm_a[j]));
          pm_b[j] = fmaf(x[s][1], m0, fmaf(x[s][3], m1, pm_b[j]));
          const uint32_t b0 = movmatrix_trans(w[s][j][0]), b1 = movmatrix_trans(w[s][j][1]);
          const uint32_t xl = __byte_perm(v00[j], v01[j], 0x5410), yl = __byte_perm(v00[j], v01[j], 0x7632);
          const uint32_t xh = __byte_perm(v10[j], v11[j], 0x5410), yh = __byte_perm(v10[j], v11[j], 0x7632);
          // channels 0, 1 of the lane's word by their own codes, 2, 3 by whole bytes c + 16 c' (less those of 0, 1 at the end); 4 .. 7 alike
          const uint32_t xl8 = __byte_perm(xl, 0u, 0x4341), yl8 = __byte_perm(yl, 0u, 0x4341);
          const uint32_t xh8 = __byte_perm(xh, 0u, 0x4341), yh8 = __byte_perm(yh, 0u, 0x4341);
          mma_f16_16816(o[4 * j], xl & LO, yl & LO, xh & LO, yh & LO, b0, b1);
          mma_f16_16816(o[4 * j + 1], xl & BYTE, yl & BYTE, xh & BYTE, yh & BYTE, b0, b1);
          mma_f16_16816(o[4 * j + 2], xl8 & LO, yl8 & LO, xh8 & LO, yh8 & LO, b0, b1);
          mma_f16_16816(o[4 * j + 3], xl8, yl8, xh8, yh8, b0, b1);
        }
      }
    }

    // ---- the end of the row, or of this warp's part of it; the next row's q is on its way meanwhile ------------------------------------
    const int b = cs_s[warp].b, h = cs_s[warp].h;
    __syncwarp();
    if (t < w1) {
      Walk to = cs_s[warp];
      to.i = to.count - 1;
      to.next(p);
      ask_q(to.b, to.h);
      __syncwarp();
      if (lane == 0) cs_s[warp] = to;
      __syncwarp();
    }
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      l_a += __shfl_xor_sync(FULL, l_a, off);
      l_b += __shfl_xor_sync(FULL, l_b, off);
#pragma unroll
      for (int j = 0; j < GRP; ++j) {
        pm_a[j] += __shfl_xor_sync(FULL, pm_a[j], off);
        pm_b[j] += __shfl_xor_sync(FULL, pm_b[j], off);
      }
    }
    const bool complete = row_t0 >= w0 && row_t1 <= w1;
    float* part = nullptr;
    if (!complete) {
      // the warp's last part can take the place of its ring, an earlier one (its first row's end) has a place of its own
      if (seg_end == w1) {
        cp_async_wait<0>();
        __syncwarp();
        part = reinterpret_cast<float*>(smem + warp * C::RING);
      } else {
        part = reinterpret_cast<float*>(smem + NW * C::RING + warp * C::PART);
      }
      if (lane == 0) {
        const int slot = seg_end == w1 ? 1 : 0;
        meta_s[warp][slot][0] = b * p.hkv + h;
        meta_s[warp][slot][1] = row_t0;
        meta_s[warp][slot][2] = row_t1;
      }
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int head = 2 * c4 + side;
      if (head >= G) continue;
      const float l = side ? l_b : l_a, m = side ? m_b : m_a;
      const float inv = l > 0.f ? (complete ? p.out_scale : 1.f) / l : 0.f;
#pragma unroll
      for (int j = 0; j < C::WV; ++j) {
        const float by = 0x1p24f * pow2_inverse(side ? up[j].y : up[j].x), by16 = by * 0.0625f;
        float y[8];                                          // channels 64 j + 8 g ..: rows g (even) and g + 8 (odd) of four tiles
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float add = side ? pm_b[j] : pm_a[j];
          const float* even = o[4 * j + (i & 2)];
          const float* at = o[4 * j + i];
          y[2 * i] = (i & 1) ? fmaf(at[side] - even[side], by16, add) * inv : fmaf(at[side], by, add) * inv;
          y[2 * i + 1] = (i & 1) ? fmaf(at[2 + side] - even[2 + side], by16, add) * inv : fmaf(at[2 + side], by, add) * inv;
        }
        if (complete) store_vec<__nv_bfloat16, 8>(p.out + b * p.out_stride + (static_cast<int64_t>(h) * G + head) * D + 64 * j + 8 * g, y);
        else store_f32<8>(part + head * D + 64 * j + 8 * g, y);
      }
      if (!complete && g == 0) lse_s[seg_end == w1 ? 1 : 0][head][warp] = l == 0.f ? -INFINITY : m + fast_log2(l);    // (NaN stays NaN)
    }
    row_t0 = row_t1;
  }
  cp_async_wait<0>();
  __syncthreads();

  // ---- parts of rows, put together --------------------------------------------------------------------------------------------------
  // The parts of a row are those of neighbouring warps, one of each: last parts, and perhaps a first part of the last of these warps.  This
  // code runs once, from a cold instruction cache and a load behind the other: one copy of it serves all jobs, and inside it what can be
  // requested at once is.
  const Decode4Share mine_s = cut_s;
  const int t0 = mine_s.t0, t1 = mine_s.t1;
  const int* meta = &meta_s[0][0][0];
  const int of_lane = lane < NW ? lane : 0;
  const int row_f = lane < NW ? meta_s[of_lane][0][0] : -1, row_l = lane < NW ? meta_s[of_lane][1][0] : -1;
  // four outputs of a row and the log2-sum-exp of their head, from the warps of the masks
  auto sum_parts = [&](uint32_t f, uint32_t l, int e, float& lse) -> float4 {
    const int head = e * 4 / D, wf = __ffs(f) - 1;           // (-1: no first part)
    const int lo = l != 0 ? __ffs(l) - 1 : 0, hi = 31 - __clz(l);            // (no last part: hi is -1)
    const float xf = wf >= 0 ? lse_s[0][head][wf] : -INFINITY;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float M = xf;
    for (int w0 = lo; w0 <= hi; w0 += 4) {
#pragma unroll
      for (int k = 0; k < 4; ++k) M = fmaxf(M, w0 + k <= hi ? lse_s[1][head][w0 + k] : -INFINITY);       // (-inf: a warp without tiles)
    }
    const float r = M == -INFINITY ? 0.f : M;
    float sum = fast_exp2(xf - r);
    if (wf >= 0) {
      const float4 y = *reinterpret_cast<const float4*>(smem + NW * C::RING + wf * C::PART + e * 16);
      acc.x = sum * y.x; acc.y = sum * y.y; acc.z = sum * y.z; acc.w = sum * y.w;
    }
    for (int w0 = lo; w0 <= hi; w0 += 4) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float x = w0 + k <= hi ? lse_s[1][head][w0 + k] : -INFINITY;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        if (x > -INFINITY) y = *reinterpret_cast<const float4*>(smem + (w0 + k) * C::RING + e * 16);
        const float a = fast_exp2(x - r);
        acc.x = fmaf(a, y.x, acc.x); acc.y = fmaf(a, y.y, acc.y); acc.z = fmaf(a, y.z, acc.z); acc.w = fmaf(a, y.w, acc.w);
        sum += a;
      }
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
    lse = sum == 0.f ? -INFINITY : M + fast_log2(sum);
    return acc;
  };
  auto put = [&](int row, int e, const float4& y, float f) {
    const int b = row / p.hkv, h = row - b * p.hkv;
    *reinterpret_cast<uint2*>(p.out + b * p.out_stride + static_cast<int64_t>(h) * G * D + e * 4) =
        make_uint2(pack_bf16(y.x * f, y.y * f), pack_bf16(y.z * f, y.w * f));
  };
  // Job 0, 1: the rows of this warp's own parts, where they end in the CTA; the warps with a part of a row share its outputs.  Job 2, 3: the
  // CTA's first and last row, where they go on in other CTAs: every warp takes D / NW channels of all heads, in every CTA alike.
  constexpr int PIECES = D / NW / 4;                         // 16-byte pieces of a head that a warp takes of such a row
  const int owned = G * PIECES, E4 = G * D / 4;
  const uint32_t cross_f = __ballot_sync(FULL, row_f >= 0 && (meta_s[of_lane][0][1] < t0 || meta_s[of_lane][0][2] > t1));
  const uint32_t cross_l = __ballot_sync(FULL, row_l >= 0 && (meta_s[of_lane][1][1] < t0 || meta_s[of_lane][1][2] > t1));
  auto piece = [&](int i) -> int { return i / PIECES * (D / 4) + warp * PIECES + i % PIECES; };   // of the share, as a piece of the row
  int mine_row = -1, mine_first = 0, mine_last = 0;          // lanes 0 and 1: the crossing rows
#pragma unroll 1
  for (int job = 0; job < 4; ++job) {
    int slot;
    if (job < 2) {
      slot = 2 * warp + job;
    } else {
      const uint32_t any = cross_f | cross_l;
      if (any == 0) return;                                  // (the whole CTA)
      const int w = job == 2 ? __ffs(any) - 1 : 31 - __clz(any);
      slot = 2 * w + (job == 2 ? (cross_f >> w & 1 ? 0 : 1) : static_cast<int>(cross_l >> w & 1));
    }
    const int row = meta[slot * 3], r0 = meta[slot * 3 + 1], r1 = meta[slot * 3 + 2];
    if (row < 0 || (job < 2 && (r0 < t0 || r1 > t1))) continue;
    if (job == 3 && row == __shfl_sync(FULL, mine_row, 0)) continue;
    const uint32_t f = __ballot_sync(FULL, row_f == row), l = __ballot_sync(FULL, row_l == row);
    int at = lane, end = owned;
    if (job < 2) {
      const int parts = __popc(f | l), mine = __popc((f | l) & ((1u << warp) - 1));
      at = mine * E4 / parts + lane; end = (mine + 1) * E4 / parts;
    } else if (lane == job - 2) {
      mine_row = row; mine_first = r0; mine_last = r1;
    }
    float* to = p.parts + (static_cast<int64_t>(cta) * 2 + (r0 <= t0 ? 0 : 1)) * decode4_part(G, D);
    for (; at < end; at += 32) {
      const int e = job < 2 ? at : piece(at);
      float lse;
      const float4 y = sum_parts(f, l, e, lse);
      if (job < 2) {
        put(row, e, y, p.out_scale);
      } else {
        *reinterpret_cast<float4*>(to + e * 4) = y;
        if (at % PIECES == 0) to[G * D + kDecode4MaxGroup * warp + at / PIECES] = lse;
      }
    }
  }
  // Of the warps with the same channels of a crossing row, the one that arrives last finds all parts of them in memory.
  __syncwarp();                                              // the lanes' parts come before the release
  const Decode4Cut cut(total_s, NW);
  int c1 = mine_s.first, parts = mine_s.parts;
  if (mine_row < 0) {
    parts = 0;
  } else {
    if (c1 < 0) {
      c1 = cut.of(mine_first);
      parts = cut.of(mine_last - 1) - c1 + 1;
    }
    int32_t* count = p.arrivals + static_cast<int64_t>(mine_row) * NW + warp;
    int prev;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(prev) : "l"(count) : "memory");
    if (prev == parts - 1) *count = 0;                       // as the next launch expects it
    else parts = 0;
  }
  __syncwarp();
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const int n = __shfl_sync(FULL, parts, i);
    if (n == 0) continue;
    const int from_cta = __shfl_sync(FULL, c1, i), row = __shfl_sync(FULL, mine_row, i), r0 = __shfl_sync(FULL, mine_first, i);
    // a lane takes a piece, or the piece of every n-th part where a warp's share leaves lanes over
    const int lanes = min(owned, 32), split = 32 / lanes, mine = lane / lanes, first = lane - mine * lanes;
    const float* head_part = p.parts + static_cast<int64_t>(from_cta) * 2 * decode4_part(G, D);
    const int64_t stride = 2 * decode4_part(G, D);
    const int late = mine_s.first >= 0 || r0 <= cut.start(from_cta) ? 0 : decode4_part(G, D);          // the first CTA's part, where the row began inside it
    for (int base = 0; base < owned; base += 32) {
      const int e = piece(base + first);
      const bool works = mine < split && base + first < owned;
      float M = -INFINITY, sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      if (works) {
        const int at_lse = G * D + kDecode4MaxGroup * warp + (base + first) / PIECES;
        constexpr int AT_ONCE = 8;                           // parts requested before the first is used
        for (int c0 = mine; c0 < n; c0 += AT_ONCE * split) {
          float lse[AT_ONCE], most = M;
          float4 v[AT_ONCE];
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) {
            const int c = c0 + k * split;
            const float* from = head_part + c * stride + (c == 0 ? late : 0);
            lse[k] = c < n ? __ldcg(from + at_lse) : -INFINITY;
            v[k] = c < n ? __ldcg(reinterpret_cast<const float4*>(from + e * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) most = fmaxf(most, lse[k]);
          const float r = most == -INFINITY ? 0.f : most, a = fast_exp2(M - r);
          acc.x *= a; acc.y *= a; acc.z *= a; acc.w *= a; sum *= a;
          M = most;
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) {
            const float f = fast_exp2(lse[k] - r);
            acc.x = fmaf(f, v[k].x, acc.x); acc.y = fmaf(f, v[k].y, acc.y); acc.z = fmaf(f, v[k].z, acc.z); acc.w = fmaf(f, v[k].w, acc.w);
            sum += f;
          }
        }
      }
      float top = M;
      for (int k = 0; k < split; ++k) top = fmaxf(top, __shfl_sync(FULL, M, first + k * lanes));
      const float a = M == -INFINITY ? 0.f : fast_exp2(M - top);
      const float4 own = make_float4(acc.x * a, acc.y * a, acc.z * a, acc.w * a);
      const float own_sum = sum * a;
      acc = own; sum = own_sum;
      for (int k = 1; k < split; ++k) {                      // (lanes of the first part add the others)
        const int from = first + k * lanes;
        acc.x += __shfl_sync(FULL, own.x, from); acc.y += __shfl_sync(FULL, own.y, from); acc.z += __shfl_sync(FULL, own.z, from);
        acc.w += __shfl_sync(FULL, own.w, from); sum += __shfl_sync(FULL, own_sum, from);
      }
      if (works && mine == 0) put(row, e, acc, sum > 0.f ? p.out_scale / sum : 0.f);
    }
  }
}

// The parts have the room that the largest head shape needs, so that the counters lie at the same place for every shape and batch: one
// workspace may serve different calls one after the other and the counters are zero between them.
constexpr size_t kDecode4Parts = sizeof(float) * kDecode4MaxCtas * 2 * decode4_part(kDecode4MaxGroup, 256);
static_assert(kDecode4Parts % 256 == 0, "the counters lie at a multiple of 256 bytes");

static size_t decode4_bytes(int64_t seqs, int hkv) {
  return kDecode4Parts + (sizeof(int32_t) * static_cast<size_t>(seqs) * hkv * kDecode4MaxWarps + 255) / 256 * 256;
}

}  // namespace mvb

extern "C" size_t mvb_decode_attn4_workspace_bytes(int max_seqs, int num_q_heads, int num_kv_heads, int head_dim) {
  if (max_seqs <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || num_q_heads % num_kv_heads != 0) return 0;
  return mvb::decode4_bytes(max_seqs, num_kv_heads);
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
  const int hkv = cache->num_kv_heads;
  if (num_q_heads % hkv != 0 || num_q_heads / hkv > kDecode4MaxGroup) return kUnsupportedShape;
  if (num_seqs == 0) return kOk;
  if (!q || !out || !cache_seqlens || !block_table || !workspace) return kInvalidArgument;
  if (q_row_stride % 8 || out_row_stride % 8 || !is_aligned(q, 16) || !is_aligned(out, 16) || !is_aligned(workspace, 256)) return kMisaligned;
  // lengths and tile numbers are 32-bit
  if (static_cast<int64_t>(table_width) * cache->block_size > 0x7fffffffLL || num_seqs > 65535) return kUnsupportedShape;
  const int64_t longest = table_width < cache->num_blocks ? table_width : cache->num_blocks;
  if (static_cast<double>(num_seqs) * hkv * (longest * (cache->block_size / 32) + 1) > 2147483000.0) return kUnsupportedShape;
  if (workspace_bytes < decode4_bytes(num_seqs, hkv)) return kScratchTooSmall;
  const float kLog2e = 1.4426950408889634f;
  Decode4Params p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.q_stride = q_row_stride; p.out = static_cast<__nv_bfloat16*>(out); p.out_stride = out_row_stride;
  p.k_codes = static_cast<const uint8_t*>(cache->k_codes); p.v_codes = static_cast<const uint8_t*>(cache->v_codes);
  p.k_affine = static_cast<const uint8_t*>(cache->k_affine); p.v_affine = static_cast<const uint8_t*>(cache->v_affine);
  p.seqlens = cache_seqlens; p.block_table = block_table; p.table_stride = table_stride; p.table_width = table_width; p.spans = spans;
  p.num_blocks = cache->num_blocks; p.by_block = FastDiv(static_cast<uint32_t>(cache->block_size));
  p.max_len = static_cast<int>(longest * cache->block_size); p.num_seqs = num_seqs; p.hkv = hkv; p.group = num_q_heads / hkv; p.block_size = cache->block_size;
  p.budget = budget; p.window_left = window_left;
  // with a cap the scores leave the sums as they are and the cap's own factors are in log2 units
  p.scale_log2 = softcap > 0.f ? scale : scale * kLog2e;
  p.cap_in = softcap > 0.f ? 2.f * kLog2e / softcap : 0.f; p.cap_log2 = softcap * kLog2e; p.out_scale = out_scale;
  p.parts = static_cast<float*>(workspace);
  p.arrivals = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + kDecode4Parts);
  p.dev_status = dev_status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int grid = sm_count() < kDecode4MaxCtas ? sm_count() : kDecode4MaxCtas;
  // Sixteen warps keep an SM's pipes busier, eight have twice the registers and are quicker from the first load to the last part (and take a
  // shorter row by themselves): eight up to 200 tiles an SM (80 of 64-wide heads), as far as the call can tell; always eight for heads of 256,
  // whose fragments need the registers.  8 heads of 128, sixteen and eight: 1 context of 700 tokens 12.9 and 10.2 us, of 40000 23.6 and 19.9, 32 of
  // 1000 23.8 and 19.8, 32 of 4000 41.3 and 39.7, 4 of 40000 48.0 and 46.5, 16 of 16000 63 and 66, 64 of 4000 63 and 66.  2 heads of 64: 1 of 40000 17.0
  // and 13.9, 32 of 4000 17.1 and 17.7, 16 of 16000 21.4 and 22.0.  Lists of spans, a run of loads more for every two tiles, half of that: 8 heads of
  // 128, 64 spans for 1 sequence 16.1 and 11.8, 16 for 48 30.4 and 27.0, 16 for 96 41.4 and 41.8, 64 for 64 77 and 86
  int64_t most = longest * cache->block_size / 32 + 1;       // tiles of a row
  if (window_left >= 0 && (static_cast<int64_t>(window_left) + 1) / 32 + 2 < most) most = (static_cast<int64_t>(window_left) + 1) / 32 + 2;
  if (spans != nullptr && static_cast<int64_t>(budget) * (kKv4Span / 32) < most) most = static_cast<int64_t>(budget) * (kKv4Span / 32);
  const bool few = static_cast<int64_t>(num_seqs) * hkv * most <= static_cast<int64_t>(sm_count()) * (cache->head_dim == 64 ? 80 : 200) / (spans != nullptr ? 2 : 1);
  auto launch = [&](auto tag, auto cap, auto warps) -> int {
    constexpr int D = decltype(tag)::value, W = decltype(warps)::value;
    using C = Decode4Cfg<D, W>;
    struct Tag {};
    const int r = opt_in_dynamic_smem<Tag>(reinterpret_cast<const void*>(&kv4_decode_kernel<D, decltype(cap)::value, W>), C::SMEM);
    if (r != kOk) return r;
    kv4_decode_kernel<D, decltype(cap)::value, W><<<grid, C::NW * 32, C::SMEM, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
  };
  auto by_cap = [&](auto tag, auto warps) -> int { return softcap > 0.f ? launch(tag, std::true_type{}, warps) : launch(tag, std::false_type{}, warps); };
  const std::integral_constant<int, 8> eight{};
  const std::integral_constant<int, 16> sixteen{};
  if (cache->head_dim == 64) return few ? by_cap(std::integral_constant<int, 64>{}, eight) : by_cap(std::integral_constant<int, 64>{}, sixteen);
  if (cache->head_dim == 128) return few ? by_cap(std::integral_constant<int, 128>{}, eight) : by_cap(std::integral_constant<int, 128>{}, sixteen);
  return by_cap(std::integral_constant<int, 256>{}, eight);
}
