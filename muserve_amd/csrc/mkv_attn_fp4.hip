// mkv_attn_fp4.hip — paged decode attention over a 4-bit pool (gfx950): rows of
// e2m1 codes and e8m0 scales (mkv_quant.h), dequantised in registers.
//
// One query token per sequence attends to the first seq_lens[b] cached tokens
// of its block table: softmax(q k^T * scale) v for each of the G query heads
// that share a KV head. A cached token and head is 2 x 136 bytes for 1024 * G
// flop, so HBM bounds the launch.
//   * Work split: the (sequence, KV head) pairs' tiles of 32 tokens (two pages)
//     form one flat list, pair after pair. Each wave of the resident grid takes
//     an equal contiguous span of it; pieces of pairs that spans cut leave
//     (max, sum, unnormalised output) and a second kernel joins them.
//   * Scores on the matrix cores (16x16x32 bf16): A = the 16 K rows of a page,
//     codes converted to bf16 with their scale (exact), B = the query heads in
//     columns n and n + 8. A column's lanes hold 8 tokens each; the maximum is
//     lazy (raised when a score passes it by 2^8), so most tiles need no
//     reduction over lanes, and each lane sums its own tokens' weights.
//   * P V on the matrix cores: A = the weights in two bf16 parts (the rows n
//     hold the upper 8 bits, the rows n + 8 the next 8: 16 bits of weight for
//     the price of rows that would be empty), B = V, 16 dims a lane. The score
//     tile's lanes already hold the A operand: the tokens' order inside the
//     product is free, so V is read in theirs.
#include <math.h>

#include "mkv_quant.h"

namespace mkv {
namespace {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4a8 __attribute__((ext_vector_type(4), aligned(8)));

constexpr int kHeadDim = 256;
constexpr int kQRow = kHeadDim * 2;
constexpr int kThreads4 = 256;
constexpr int kWaves = kThreads4 / 64;
constexpr int kTile = 32;            // tokens of a tile: two pages
constexpr int kMaxGroup = 8;         // query heads per KV head
constexpr int kMaxPairs = 4096;      // batch x KV heads
constexpr int kWgsPerCu = 2;
constexpr int kJointTiles = 8;       // tiles a pair, on average, from which spans are workgroups'
constexpr int kWidePairs = 128;      // pairs below which the merge takes 16 waves
constexpr float kRaise = 8.f;        // log2 by which a score may pass the running maximum

struct Args {
  const uint8_t* q;      // [B, Hkv * G, 256] bf16
  const uint8_t* k;      // [P, 16, Hkv, 136]
  const uint8_t* v;
  const int32_t* table;  // [B, tstride]
  const int32_t* lens;   // [B]
  uint8_t* out;          // [B, Hkv * G, 256] bf16
  int64_t* hdr;          // workspace: [0] tiles of a span
  int32_t* pre;          // [pairs + 1] each pair's first flat tile
  float* ml;             // [waves, 2, G, 2] (max, sum) of cut pairs' pieces, log2 units
  float* part;           // [waves, 2, G, 256] their unnormalised outputs
  int64_t num_pages, tstride, shared_below;
  int32_t twidth, hkv, group, max_len, pairs;
  float scale_log2;
  int32_t* err;
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Eight codes of a word times the scale, as eight bf16.
__device__ __forceinline__ u32x4 dequant8(uint32_t w, float s) {
  return u32x4{mkv_fp4_pair(w, 0, s), mkv_fp4_pair(w, 1, s), mkv_fp4_pair(w, 2, s),
               mkv_fp4_pair(w, 3, s)};
}

// A tile's cached rows, as a lane holds them: of each page the dims 32 g .. and 128 +
// 32 g .. of K token c, and the dims 16 c .. of V tokens 4 g + j. One load of V scales
// serves the page: lane c's word is of token 4 g + c % 4, the half c / 8 of its blocks.
struct Tile {
  u32x4 k[2][2];
  u32x2 ks[2];
  u32x2 v[2][4];
  uint32_t vs[2];
};

__global__ __launch_bounds__(kThreads4, 2) void attn_fp4_span_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) float piece_l[];  // [waves][G][256], then (m, l)
  __shared__ int32_t wave_tot[kWaves];
  __shared__ int32_t start_l[kWaves][2];  // (pair, its first tile) that a span starts in
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t cap = (int64_t)a.twidth * 16 < a.max_len ? (int64_t)a.twidth * 16 : a.max_len;
  // a pair's cached tokens, cut to the table and the launch's bound
  auto length_of = [&](int pr) __attribute__((always_inline)) {
    const int64_t len = ld_const(a.lens + pr / a.hkv);
    return (int32_t)(len < 0 ? 0 : (len > cap ? cap : len));
  };
  // exclusive prefix of the tile counts of 256 pairs from `base` on, behind `before`;
  // the round's total goes to `round`
  auto scan = [&](int base, int32_t before, int32_t& cnt, int32_t& round)
      __attribute__((always_inline)) {
    const int pr = base + tid;
    cnt = pr < a.pairs ? (length_of(pr) + kTile - 1) / kTile : 0;
    int32_t incl = cnt;
#pragma unroll
    for (int dd = 1; dd < 64; dd <<= 1) {
      const int32_t o = __shfl_up(incl, dd);
      if (lane >= dd) incl += o;
    }
    __syncthreads();  // wave_tot's earlier readers are done
    if (lane == 63) wave_tot[wave] = incl;
    __syncthreads();
    int32_t at = before + incl - cnt;
    round = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      at += w < wave ? wave_tot[w] : 0;
      round += wave_tot[w];
    }
    return at;
  };
  int32_t T = 0, cnt, round, at = 0;
  for (int base = 0; base < a.pairs; base += kThreads4) {
    at = scan(base, T, cnt, round);
    T += round;
  }
  if (T == 0) {
    if (blockIdx.x == 0) {
      for (int p = tid; p <= a.pairs; p += kThreads4) a.pre[p] = 0;
      for (int p = tid; p < a.pairs; p += kThreads4)
        if (ld_const(a.lens + p / a.hkv) < 0) raise_err(a.err, MKV_DEVERR_TABLE);
    }
    return;
  }
  // Spans: by workgroup, its waves taking the tiles in turn and joining their pieces in
  // LDS, where a pair has enough tiles to keep them busy; else by wave.
  const bool joint = T >= kJointTiles * a.pairs;
  const int32_t step = joint ? kWaves : 1;
  const int32_t units = (int32_t)gridDim.x * (joint ? 1 : kWaves);
  int32_t S = (T + units - 1) / units;
  S = S < step ? step : S;
  const int32_t unit = joint ? (int32_t)blockIdx.x : (int32_t)blockIdx.x * kWaves + wave;
  // the pairs that this workgroup's spans start in (and, by workgroup 0, all prefixes for
  // the merge kernel); a round's prefix is still held where there is one round
  {
    const int32_t first = joint ? (int32_t)blockIdx.x : (int32_t)blockIdx.x * kWaves;
    int32_t before = 0;
    for (int base = 0; base < a.pairs; base += kThreads4) {
      if (a.pairs > kThreads4) {
        at = scan(base, before, cnt, round);
        before += round;
      }
      const int pr = base + tid;
      if (pr < a.pairs) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const int64_t s = (int64_t)(first + w) * S;
          if ((w == 0 || !joint) && s >= at && s < at + cnt) {
            start_l[w][0] = pr;
            start_l[w][1] = at;
          }
        }
        if (blockIdx.x == 0) {
          a.pre[pr] = at;
          const int64_t len = ld_const(a.lens + pr / a.hkv);
          if ((len > cap || len < 0) && pr % a.hkv == 0) raise_err(a.err, MKV_DEVERR_TABLE);
        }
      }
    }
    if (blockIdx.x == 0 && tid == 0) {
      a.pre[a.pairs] = T;
      a.hdr[0] = S;
    }
    __syncthreads();
  }
  const int64_t s64 = (int64_t)unit * S;
  if (s64 >= T) return;  // (joint: the whole workgroup)
  const int32_t s0 = (int32_t)s64, s1 = s64 + S < T ? (int32_t)s64 + S : T;
  const int32_t w0 = joint ? wave : 0;  // the wave takes the span's tiles w0, w0 + step, ..

  const int c = lane & 15, g = lane >> 4;  // row / column and quad of a matrix operand
  const int head = c & 7;
  const uint32_t low_mask = c < 8 ? 0u : 0xffff0000u;  // what the lane takes off a weight
  const int64_t row_bytes = (int64_t)a.hkv * kFp4Row;
  const int64_t page_bytes = 16 * row_bytes;
  const uint32_t koff = (uint32_t)(c * row_bytes);
  const uint32_t voff = (uint32_t)(4 * g * row_bytes), vstep = (uint32_t)row_bytes;
  const uint32_t vsoff = (uint32_t)((4 * g + (c & 3)) * row_bytes) + kFp4Codes + 4 * (c >> 3);
  const uint32_t vshift = 8 * ((c >> 1) & 3), kshift = 8 * g;

  // a pair as the walk over the span has it
  struct Pair {
    int32_t p, pre0, pre1, len;
  };
  auto next_pair = [&](Pair& x) __attribute__((always_inline)) {  // the next one with tiles
    do {
      ++x.p;
      x.len = __builtin_amdgcn_readfirstlane(length_of(x.p));
      x.pre0 = x.pre1;
      x.pre1 += (x.len + kTile - 1) / kTile;
    } while (x.pre1 == x.pre0);
  };
  Pair ahead;  // of the tile whose page ids are read next
  {
    const int w = joint ? 0 : wave;
    ahead.p = __builtin_amdgcn_readfirstlane(start_l[w][0]);
    ahead.pre0 = __builtin_amdgcn_readfirstlane(start_l[w][1]);
    ahead.len = __builtin_amdgcn_readfirstlane(length_of(ahead.p));
    ahead.pre1 = ahead.pre0 + (ahead.len + kTile - 1) / kTile;
  }
  Pair cur = ahead;
  // A tile's rows are loaded while the one before it is computed, and its page ids a tile
  // earlier still: the rows' loads wait for them.
  struct Pages {
    int32_t id[2], left[2], hk;  // left: the page's tokens and those behind it
  };
  int32_t fa = s0 + w0;
  auto read_ids = [&](Pages& x) __attribute__((always_inline)) {  // of tile fa
    if (fa >= s1) {  // behind the span: a page that is in the caches, no token of it
      x.id[0] = x.id[1] = x.left[0] = x.left[1] = x.hk = 0;
      return;
    }
    while (fa >= ahead.pre1) next_pair(ahead);
    const int b = ahead.p / a.hkv;
    const int32_t tok0 = (fa - ahead.pre0) * kTile;
    const int32_t* ids = a.table + (int64_t)b * a.tstride + tok0 / 16;
    x.hk = ahead.p - b * a.hkv;
    x.left[0] = ahead.len - tok0;
    x.left[1] = x.left[0] - 16;
    x.id[0] = ld_const(ids);
    x.id[1] = ld_const(ids + (x.left[1] > 0 ? 1 : 0));
    fa += step;
  };
  auto load = [&](Tile& t, const Pages& x, int32_t (&valid)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int32_t left = x.left[i] < 0 ? 0 : (x.left[i] > 16 ? 16 : x.left[i]);
      int32_t id = x.id[i];
      if (id < 0 || id >= a.num_pages) {  // no token of a page id outside the pool
        if (lane == 0 && left > 0) raise_err(a.err, MKV_DEVERR_PAGE);
        id = 0;
        left = 0;
      }
      valid[i] = left;
      const int64_t base = id * page_bytes + x.hk * kFp4Row;
      const uint8_t* kp = a.k + base;
      const uint8_t* vp = a.v + base;
      t.k[i][0] = *reinterpret_cast<const u32x4a8*>(kp + (koff + 16 * g));
      t.k[i][1] = *reinterpret_cast<const u32x4a8*>(kp + (koff + 16 * g + 64));
      t.ks[i] = *reinterpret_cast<const u32x2*>(kp + (koff + kFp4Codes));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        t.v[i][j] = *reinterpret_cast<const u32x2*>(vp + (voff + j * vstep + 8 * c));
      t.vs[i] = *reinterpret_cast<const uint32_t*>(vp + vsoff);
    }
  };

  u32x4 qb[8];
  f32x4 acc[16];
  float m_run, l_run;
  auto compute = [&](const Tile& t, const int32_t (&valid)[2]) __attribute__((always_inline)) {
    // scores: lane (c, g) gets tokens 4 g + j of each page, for head c & 7
    float sv[8], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x4 sc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float scale = fp4_scale((t.ks[i][h] >> kshift) & 255u);
#pragma unroll
        for (int s = 0; s < 4; ++s)
          sc = mfma(dequant8(t.k[i][h][s], scale), qb[4 * h + s], sc);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sv[4 * i + j] = 4 * g + j < valid[i] ? sc[j] * a.scale_log2 : -INFINITY;
        mx = fmaxf(mx, sv[4 * i + j]);
      }
    }
    if (__builtin_amdgcn_ballot_w64(mx > m_run + kRaise) != 0) {
      const float top = over_rows<4>(mx, [](float x, float y) { return fmaxf(x, y); });
      const float m_new = fmaxf(m_run, top);
      const float alpha = m_run == -INFINITY ? 0.f : exp2_fast(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
      // output rows 4 g + i belong to head (4 g + i) & 7
      float al[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) al[i] = __shfl(alpha, (4 * g + i) & 7);
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] *= al[i];
    }
    const float m_ref = m_run == -INFINITY ? 0.f : m_run;
    u32x4 pa;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float p0 = exp2_fast(sv[j] - m_ref), p1 = exp2_fast(sv[j + 1] - m_ref);
      l_run += p0 + p1;
      // upper 8 bits of the weight in rows below 8, what is left of it in the others
      const uint32_t x0 = f32_bits(p0 - bits_f32(f32_bits(p0) & low_mask));
      const uint32_t x1 = f32_bits(p1 - bits_f32(f32_bits(p1) & low_mask));
      pa[j / 2] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
    }
    u32x2 v[8];
    float vsc[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w[4] = {lane_of<0x00>(t.vs[i]), lane_of<0x55>(t.vs[i]), lane_of<0xaa>(t.vs[i]),
                             lane_of<0xff>(t.vs[i])};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[4 * i + j] = t.v[i][j];
        vsc[4 * i + j] = fp4_scale((w[j] >> vshift) & 255u);
      }
    }
    if (valid[0] < 16 || valid[1] < 16) {  // rows that hold anything: zeros
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool ok = 4 * g + (j & 3) < valid[j >> 2];
        v[j] = ok ? v[j] : u32x2{0u, 0u};
        vsc[j] = ok ? vsc[j] : 1.f;
      }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      // dims 8 w + 2 e and + 1 of the lane's 16, of its 8 tokens: pairs of dims to pairs of tokens
#define MKV_PV(e)                                                                              \
  {                                                                                            \
    u32x4 lo, hi;                                                                              \
    _Pragma("unroll") for (int j = 0; j < 4; ++j) {                                            \
      const uint32_t x0 = mkv_fp4_pair(v[2 * j][w], e, vsc[2 * j]);                            \
      const uint32_t x1 = mkv_fp4_pair(v[2 * j + 1][w], e, vsc[2 * j + 1]);                    \
      lo[j] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);                                      \
      hi[j] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);                                      \
    }                                                                                          \
    acc[8 * w + 2 * e] = mfma(pa, lo, acc[8 * w + 2 * e]);                                     \
    acc[8 * w + 2 * e + 1] = mfma(pa, hi, acc[8 * w + 2 * e + 1]);                             \
  }
      MKV_PV(0) MKV_PV(1) MKV_PV(2) MKV_PV(3)
#undef MKV_PV
    }
  };

  Tile t;
  Pages pages;
  int32_t valid[2];
  int32_t f = s0 + w0;  // the wave's next tile
  read_ids(pages);
  load(t, pages, valid);
  read_ids(pages);
  for (;;) {            // the span's pairs
    const int32_t end = cur.pre1 < s1 ? cur.pre1 : s1;
#pragma unroll
    for (int s = 0; s < 8; ++s) {  // the dims of K's operand: 32 g + 8 s, 128 + 32 g + 8 (s - 4)
      const int dim = 32 * g + 8 * (s & 3) + 128 * (s >> 2);
      qb[s] = head < a.group
                  ? ld16(a.q + ((int64_t)cur.p * a.group + head) * kQRow + 2 * dim)
                  : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run = -INFINITY;
    l_run = 0.f;
    while (f < end) {
      Tile next;
      int32_t next_valid[2];
      load(next, pages, next_valid);
      read_ids(pages);
      compute(t, valid);
      t = next;
      valid[0] = next_valid[0];
      valid[1] = next_valid[1];
      f += step;
    }
    // the pair's piece in this span: the quads' sums, and the weights' two parts
    const float l = over_rows<4>(l_run, [](float x, float y) { return x + y; });
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] += __shfl_xor(acc[j][i], 32);
    const bool whole = cur.pre0 >= s0 && cur.pre1 <= s1;
    // (cut pairs: the span's first goes to slot 0, its last to slot 1)
    const int64_t slot = ((int64_t)unit * 2 + (cur.pre0 <= s0 ? 0 : 1)) * a.group;
    uint8_t* out = a.out + (int64_t)cur.p * a.group * kQRow;
    if (!joint) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int h = 4 * g + i;
        const float L = __shfl(l, h & 7), M = __shfl(m_run, h & 7);
        if (h >= a.group) continue;  // (rows 8 and up are the other part)
        if (whole) {
          const float inv = 1.f / L;
          uint32_t o[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            o[j] = L == 0.f ? 0u : pack_bf16(acc[2 * j][i] * inv, acc[2 * j + 1][i] * inv);
          st16(out + h * kQRow + c * 32, u32x4{o[0], o[1], o[2], o[3]});
          st16(out + h * kQRow + c * 32 + 16, u32x4{o[4], o[5], o[6], o[7]});
        } else {
          float* dst = a.part + (slot + h) * kHeadDim + c * 16;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<f32x4*>(dst + 4 * j) = f32x4{acc[4 * j][i], acc[4 * j + 1][i],
                                                           acc[4 * j + 2][i], acc[4 * j + 3][i]};
          if (c == 0) {
            a.ml[(slot + h) * 2] = M;
            a.ml[(slot + h) * 2 + 1] = L;
          }
        }
      }
    } else {
      float* ml = piece_l + kWaves * a.group * kHeadDim;  // [waves][G][2]
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int h = 4 * g + i;
        if (h >= a.group) continue;
        float* dst = piece_l + (wave * a.group + h) * kHeadDim + c * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f32x4*>(dst + 4 * j) = f32x4{acc[4 * j][i], acc[4 * j + 1][i],
                                                         acc[4 * j + 2][i], acc[4 * j + 3][i]};
      }
      if (lane < a.group) {
        ml[(wave * a.group + lane) * 2] = m_run;
        ml[(wave * a.group + lane) * 2 + 1] = l;
      }
      __syncthreads();
      for (int h = 0; h < a.group; ++h) {  // a thread per dim
        float M = -INFINITY, O = 0.f, L = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, ml[(w * a.group + h) * 2]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float m = ml[(w * a.group + h) * 2];
          // (a wave without a score: 1, so that a NaN of its sums stays)
          const float e = m == -INFINITY ? 1.f : exp2_fast(m - M);
          O += e * piece_l[(w * a.group + h) * kHeadDim + tid];
          L += e * ml[(w * a.group + h) * 2 + 1];
        }
        if (whole) {
          reinterpret_cast<uint16_t*>(out + h * kQRow)[tid] =
              f32_to_bf16_rne(L == 0.f ? 0.f : O / L);
        } else {
          a.part[(slot + h) * kHeadDim + tid] = O;
          if (tid == 0) {
            a.ml[(slot + h) * 2] = M;
            a.ml[(slot + h) * 2 + 1] = L;
          }
        }
      }
      __syncthreads();  // the pieces are read before the next pair's
    }
    if (end == s1) return;
    next_pair(cur);
  }
}

// Joins the pieces of one (pair, query head) that spans cut, and writes the zeros of an
// empty pair. Wave w takes the pieces w, w + WAVES, .., four dims a lane, BATCH of them
// in flight; the waves' sums are joined in LDS. WAVES is 16 where few pairs leave the
// CUs idle and have many pieces, else 4.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attn_fp4_merge_kernel(Args a) {
  constexpr int BATCH = 8;
  __shared__ __attribute__((aligned(16))) float wave_o[WAVES][kHeadDim];
  __shared__ float wave_ml[WAVES][2];
  const int pr = blockIdx.x / a.group, h = blockIdx.x % a.group;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t span = ld_const(a.hdr);  // (loaded beside the pair's bounds)
  const int32_t p0 = ld_const(a.pre + pr), p1 = ld_const(a.pre + pr + 1);
  asm volatile("" ::"s"(span));
  uint16_t* out = reinterpret_cast<uint16_t*>(a.out + ((int64_t)pr * a.group + h) * kQRow);
  if (p1 <= p0) {
    if (tid < kHeadDim) out[tid] = 0;
    return;
  }
  const uint32_t S = (uint32_t)span;
  const uint32_t u0 = (uint32_t)p0 / S, u1 = (uint32_t)(p1 - 1) / S;
  if (u0 == u1) return;  // written with its span
  const int n = (int)(u1 - u0 + 1);
  auto at_of = [&](int i) __attribute__((always_inline)) {
    const int slot = i == 0 && (uint32_t)p0 != u0 * S ? 1 : 0;
    return ((int64_t)(u0 + i) * 2 + slot) * a.group + h;
  };
  float m_run = -INFINITY, l_run = 0.f;
  f32x4 o_run = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i0 = wave; i0 < n; i0 += WAVES * BATCH) {
    const int mine = i0 + WAVES * (lane & (BATCH - 1));
    const float2 ml =
        *reinterpret_cast<const float2*>(a.ml + at_of(mine < n ? mine : n - 1) * 2);
    f32x4 x[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int i = i0 + WAVES * u;
      if (i < n) x[u] = *reinterpret_cast<const f32x4*>(a.part + at_of(i) * kHeadDim + 4 * lane);
    }
    float m[BATCH], mb = m_run;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      m[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ml.x), u));
      if (i0 + WAVES * u < n) mb = fmaxf(mb, m[u]);
    }
    const float alpha = m_run == -INFINITY ? 1.f : exp2_fast(m_run - mb);
    o_run *= alpha;
    l_run *= alpha;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      if (i0 + WAVES * u >= n) break;
      const float e = m[u] == -INFINITY ? 1.f : exp2_fast(m[u] - mb);
      const float l =
          __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ml.y), u));
#pragma unroll
      for (int d = 0; d < 4; ++d) o_run[d] += e * x[u][d];
      l_run += e * l;
    }
    m_run = mb;
  }
  *reinterpret_cast<f32x4*>(&wave_o[wave][4 * lane]) = o_run;
  if (lane == 0) {
    wave_ml[wave][0] = m_run;
    wave_ml[wave][1] = l_run;
  }
  __syncthreads();
  if (tid >= kHeadDim) return;
  float M = -INFINITY, O = 0.f, L = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) M = fmaxf(M, wave_ml[w][0]);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const float e = wave_ml[w][0] == -INFINITY ? 1.f : exp2_fast(wave_ml[w][0] - M);
    O += e * wave_o[w][tid];
    L += e * wave_ml[w][1];
  }
  out[tid] = f32_to_bf16_rne(L == 0.f ? 0.f : O / L);
}

struct WsLayout {
  int64_t pre, ml, part, total;
};
WsLayout ws_layout(int64_t pairs, int64_t group) {
  const int64_t waves = (int64_t)device_cus() * kWgsPerCu * kWaves;
  WsLayout w;
  w.pre = 256;
  w.ml = w.pre + ((pairs + 1) * 4 + 255) / 256 * 256;
  w.part = w.ml + waves * 2 * group * 2 * 4;
  w.total = w.part + waves * 2 * group * kHeadDim * 4;
  return w;
}

bool shape_ok(int32_t batch, int32_t hkv, int32_t hq) {
  if (batch < 0 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || hq / hkv > kMaxGroup) return false;
  return (int64_t)batch * hkv <= kMaxPairs;
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" int64_t mkv_decode_attention_fp4_workspace_bytes(int32_t batch, int32_t num_kv_heads,
                                                            int32_t num_q_heads) {
  if (!shape_ok(batch, num_kv_heads, num_q_heads)) return -1;
  return ws_layout((int64_t)batch * num_kv_heads, num_q_heads / num_kv_heads).total;
}

extern "C" int mkv_decode_attention_fp4(const void* q, const void* k_cache, const void* v_cache,
                                        int64_t num_pages, int64_t shared_pages,
                                        int32_t num_kv_heads, int32_t num_q_heads,
                                        int32_t head_dim, const int32_t* page_table,
                                        int64_t table_stride, int32_t table_width,
                                        const int32_t* seq_lens, int32_t batch,
                                        int32_t max_seq_len, float softmax_scale, void* out,
                                        void* workspace, int64_t workspace_bytes, int32_t* err,
                                        void* stream) {
  static const char* fn = "mkv_decode_attention_fp4";
  clear_error();
  MKV_REQUIRE(batch >= 0 && num_pages > 0 && num_kv_heads > 0 && num_q_heads > 0 &&
                  table_width >= 0 && table_stride >= table_width && max_seq_len >= 0 &&
                  shared_pages >= 0,
              MKV_E_INVALID, "%s: bad sizes", fn);
  MKV_REQUIRE(head_dim == kHeadDim, MKV_E_UNSUPPORTED, "%s: head_dim %d unsupported (256)", fn,
              head_dim);
  const int32_t group = num_q_heads / num_kv_heads;
  MKV_REQUIRE(group * num_kv_heads == num_q_heads && group <= kMaxGroup, MKV_E_UNSUPPORTED,
              "%s: %d query heads on %d KV heads unsupported (1 to 8 for each)", fn, num_q_heads,
              num_kv_heads);
  if (batch == 0) return MKV_OK;
  MKV_REQUIRE(q && k_cache && v_cache && page_table && seq_lens && out && err, MKV_E_INVALID,
              "%s: null pointer", fn);
  MKV_REQUIRE(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out),
              MKV_E_ALIGN, "%s: q, caches and out must be 16-byte aligned", fn);
  MKV_REQUIRE((int64_t)batch * num_kv_heads <= kMaxPairs, MKV_E_UNSUPPORTED,
              "%s: batch x KV heads above %d", fn, kMaxPairs);
  MKV_REQUIRE(max_seq_len <= (1 << 24), MKV_E_UNSUPPORTED, "%s: max_seq_len above 2^24", fn);
  // the tiles of all pairs are counted in 32 bits
  MKV_REQUIRE((int64_t)batch * num_kv_heads * (((int64_t)max_seq_len + 15) / 16) < (1ll << 31),
              MKV_E_UNSUPPORTED, "%s: batch x KV heads x pages above 2^31", fn);
  const int32_t pairs = batch * num_kv_heads;
  const WsLayout L = ws_layout(pairs, group);
  MKV_REQUIRE(workspace && workspace_bytes >= L.total && aligned16(workspace), MKV_E_INVALID,
              "%s: workspace of %lld bytes (16-byte aligned) required", fn, (long long)L.total);
  Args a;
  a.q = static_cast<const uint8_t*>(q);
  a.k = static_cast<const uint8_t*>(k_cache);
  a.v = static_cast<const uint8_t*>(v_cache);
  a.table = page_table;
  a.lens = seq_lens;
  a.out = static_cast<uint8_t*>(out);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.hdr = reinterpret_cast<int64_t*>(ws);
  a.pre = reinterpret_cast<int32_t*>(ws + L.pre);
  a.ml = reinterpret_cast<float*>(ws + L.ml);
  a.part = reinterpret_cast<float*>(ws + L.part);
  a.num_pages = num_pages;
  a.tstride = table_stride;
  a.shared_below = shared_pages;
  a.twidth = table_width;
  a.hkv = num_kv_heads;
  a.group = group;
  a.max_len = max_seq_len;
  a.pairs = pairs;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.err = err;
  const hipStream_t st = as_stream(stream);
  const size_t lds = (size_t)kWaves * group * (kHeadDim + 2) * 4;
  hipLaunchKernelGGL(attn_fp4_span_kernel, dim3((unsigned)(device_cus() * kWgsPerCu)),
                     dim3(kThreads4), lds, st, a);
  if (pairs < kWidePairs)
    hipLaunchKernelGGL(attn_fp4_merge_kernel<16>, dim3((unsigned)(pairs * group)), dim3(16 * 64), 0,
                       st, a);
  else
    hipLaunchKernelGGL(attn_fp4_merge_kernel<4>, dim3((unsigned)(pairs * group)), dim3(4 * 64), 0,
                       st, a);
  return check_launch(fn);
}
