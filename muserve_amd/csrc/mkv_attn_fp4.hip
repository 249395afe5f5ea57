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
constexpr int kMaxPairs = 4096;      // batch x KV heads whose prefix fits in LDS
constexpr int kWgsPerCu = 2;
constexpr float kRaise = 8.f;        // log2 by which a score may pass the running maximum

struct Args {
  const uint8_t* q;      // [B, Hkv * G, 256] bf16
  const uint8_t* k;      // [P, 16, Hkv, 136]
  const uint8_t* v;
  const int32_t* table;  // [B, tstride]
  const int32_t* lens;   // [B]
  uint8_t* out;          // [B, Hkv * G, 256] bf16
  int64_t* hdr;          // workspace: [0] tiles per wave
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

// A tile's cached rows, as a lane holds them: of each page 64 dims of K token r
// (dims 64 g ..), and 16 dims (16 c ..) of V tokens 4 g + j.
struct Tile {
  u32x4 k[2][2];
  uint32_t ks[2];     // K scale bytes of the lane's two blocks
  u32x2 v[2][4];
  uint32_t vs[2][4];  // V scale byte
};

__global__ __launch_bounds__(kThreads4, 2) void attn_fp4_span_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) int32_t lds[];
  __shared__ int32_t wave_tot[kWaves];
  int32_t* pre_l = lds;                    // [pairs + 1]
  int32_t* len_l = pre_l + (a.pairs + 1);  // [pairs]
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // lengths (cut to the table and the launch's bound) and the exclusive prefix of
  // the pairs' tile counts
  const int64_t cap = (int64_t)a.twidth * 16 < a.max_len ? (int64_t)a.twidth * 16 : a.max_len;
  int32_t total = 0;
  for (int base = 0; base < a.pairs; base += kThreads4) {
    const int pr = base + tid;
    int32_t cnt = 0;
    if (pr < a.pairs) {
      int64_t len = ld_const(a.lens + pr / a.hkv);
      if (len > cap || len < 0) {
        if (blockIdx.x == 0 && pr % a.hkv == 0) raise_err(a.err, MKV_DEVERR_TABLE);
        len = len < 0 ? 0 : cap;
      }
      len_l[pr] = (int32_t)len;
      cnt = (int32_t)((len + kTile - 1) / kTile);
    }
    int32_t incl = cnt;
#pragma unroll
    for (int dd = 1; dd < 64; dd <<= 1) {
      const int32_t o = __shfl_up(incl, dd);
      if (lane >= dd) incl += o;
    }
    if (lane == 63) wave_tot[wave] = incl;
    __syncthreads();
    int32_t at = total + incl - cnt, round = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      at += w < wave ? wave_tot[w] : 0;
      round += wave_tot[w];
    }
    if (pr < a.pairs) pre_l[pr] = at;
    total += round;
    __syncthreads();
  }
  if (tid == 0) pre_l[a.pairs] = total;
  __syncthreads();
  const int64_t T = total;
  const int64_t W = (int64_t)gridDim.x * kWaves;
  const int64_t S = (T + W - 1) / W;
  if (blockIdx.x == 0) {  // for the merge kernel
    for (int p = tid; p <= a.pairs; p += kThreads4) a.pre[p] = pre_l[p];
    if (tid == 0) a.hdr[0] = S;
  }
  const int64_t gw = (int64_t)blockIdx.x * kWaves + wave;
  const int64_t s0 = gw * S < T ? gw * S : T;
  const int64_t s1 = s0 + S < T ? s0 + S : T;
  if (s0 >= s1) return;  // no barrier follows

  // the pair that holds flat tile f: the last pair p with pre[p] <= f (empty pairs
  // share their successor's prefix, so it is never empty)
  auto pair_of = [&](int64_t f) __attribute__((always_inline)) {
    int lo = 0, hi = a.pairs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pre_l[mid] <= f) lo = mid; else hi = mid - 1;
    }
    return __builtin_amdgcn_readfirstlane(lo);
  };
  const int c = lane & 15, g = lane >> 4;  // row / column and quad of a matrix operand
  const int head = c & 7;
  const uint32_t low_mask = c < 8 ? 0u : 0xffff0000u;  // what the lane takes off a weight
  const int64_t row_bytes = (int64_t)a.hkv * kFp4Row;
  const int64_t page_bytes = 16 * row_bytes;

  int p = pair_of(s0);
  int64_t pre0 = __builtin_amdgcn_readfirstlane(pre_l[p]);
  int64_t pre1 = __builtin_amdgcn_readfirstlane(pre_l[p + 1]);
  int32_t len = __builtin_amdgcn_readfirstlane(len_l[p]);
  u32x4 qb[8];
  f32x4 acc[16];
  float m_run = -INFINITY, l_run = 0.f;
  bool first = true;

  for (int64_t f = s0; f < s1; ++f) {
    if (first) {
#pragma unroll
      for (int s = 0; s < 8; ++s)  // dims 64 g + 8 s .. + 7 of the head
        qb[s] = head < a.group
                    ? ld16(a.q + ((int64_t)p * a.group + head) * kQRow + g * 128 + s * 16)
                    : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_run = -INFINITY;
      l_run = 0.f;
    }
    const int b = p / a.hkv, hk = p - b * a.hkv;
    const int32_t tok0 = (int32_t)(f - pre0) * kTile;
    // valid tokens of the tile's two pages; none of a page id outside the pool
    int32_t valid[2];
    Tile t;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int32_t left = len - tok0 - 16 * i;
      left = left < 0 ? 0 : (left > 16 ? 16 : left);
      int32_t pid = 0;
      if (left > 0) {
        pid = ld_const(a.table + (int64_t)b * a.tstride + tok0 / 16 + i);
        if (pid < 0 || pid >= a.num_pages) {
          if (lane == 0) raise_err(a.err, MKV_DEVERR_PAGE);
          pid = 0;
          left = 0;
        }
      }
      valid[i] = left;
      const int64_t base = pid * page_bytes + hk * kFp4Row;
      const uint8_t* kr = a.k + base + c * row_bytes;
      t.k[i][0] = *reinterpret_cast<const u32x4a8*>(kr + 32 * g);
      t.k[i][1] = *reinterpret_cast<const u32x4a8*>(kr + 32 * g + 16);
      t.ks[i] = *reinterpret_cast<const uint16_t*>(kr + kFp4Codes + 2 * g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t* vr = a.v + base + (4 * g + j) * row_bytes;
        t.v[i][j] = *reinterpret_cast<const u32x2*>(vr + 8 * c);
        t.vs[i][j] = vr[kFp4Codes + c / 2];
      }
    }
    // scores: lane (c, g) gets tokens 4 g + i of each page, for head c & 7
    float sv[8], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x4 sc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 8; ++s)
        sc = mfma(dequant8(t.k[i][s >> 2][s & 3], fp4_scale((t.ks[i] >> (8 * (s >> 2))) & 255u)),
                  qb[s], sc);
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
    if (valid[0] < 16 || valid[1] < 16) {  // rows that hold anything: zeros
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool ok = 4 * g + j < valid[i];
          t.v[i][j] = ok ? t.v[i][j] : u32x2{0u, 0u};
          t.vs[i][j] = ok ? t.vs[i][j] : 127u;
        }
    }
    float vsc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) vsc[j] = fp4_scale(t.vs[j >> 2][j & 3]);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      u32x4 x[8];  // dims 8 w .. + 7 of the lane's 16, of its 8 tokens
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = dequant8(t.v[j >> 2][j & 3][w], vsc[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u32x4 lo, hi;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo[j] = __builtin_amdgcn_perm(x[2 * j + 1][e], x[2 * j][e], 0x05040100u);
          hi[j] = __builtin_amdgcn_perm(x[2 * j + 1][e], x[2 * j][e], 0x07060302u);
        }
        acc[8 * w + 2 * e] = mfma(pa, lo, acc[8 * w + 2 * e]);
        acc[8 * w + 2 * e + 1] = mfma(pa, hi, acc[8 * w + 2 * e + 1]);
      }
    }
    first = f + 1 == pre1 || f + 1 == s1;
    if (!first) continue;
    // the pair's piece in this span: the quads' sums, and the weights' two parts
    const float l = over_rows<4>(l_run, [](float x, float y) { return x + y; });
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] += __shfl_xor(acc[j][i], 32);
    const bool whole = pre0 >= s0 && pre1 <= s1;
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
        uint8_t* dst = a.out + ((int64_t)p * a.group + h) * kQRow + c * 32;
        st16(dst, u32x4{o[0], o[1], o[2], o[3]});
        st16(dst + 16, u32x4{o[4], o[5], o[6], o[7]});
      } else {
        // the span's first pair goes to slot 0, its last pair to slot 1
        const int64_t at = (gw * 2 + (pre0 <= s0 ? 0 : 1)) * a.group + h;
        float* dst = a.part + at * kHeadDim + c * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f32x4*>(dst + 4 * j) = f32x4{acc[4 * j][i], acc[4 * j + 1][i],
                                                         acc[4 * j + 2][i], acc[4 * j + 3][i]};
        if (c == 0) {
          a.ml[at * 2] = M;
          a.ml[at * 2 + 1] = L;
        }
      }
    }
    if (f + 1 < s1) {
      p = pair_of(f + 1);
      pre0 = __builtin_amdgcn_readfirstlane(pre_l[p]);
      pre1 = __builtin_amdgcn_readfirstlane(pre_l[p + 1]);
      len = __builtin_amdgcn_readfirstlane(len_l[p]);
    }
  }
}

// Joins the pieces of one (pair, query head) that spans cut, and writes the zeros
// of an empty pair: a thread per dim, the pieces in order.
__global__ __launch_bounds__(kHeadDim) void attn_fp4_merge_kernel(Args a) {
  const int pr = blockIdx.x / a.group, h = blockIdx.x % a.group;
  const int tid = threadIdx.x;
  const int32_t p0 = ld_const(a.pre + pr), p1 = ld_const(a.pre + pr + 1);
  uint16_t* out = reinterpret_cast<uint16_t*>(a.out + ((int64_t)pr * a.group + h) * kQRow);
  if (p1 <= p0) {
    out[tid] = 0;
    return;
  }
  const uint32_t S = (uint32_t)ld_const(a.hdr);
  const uint32_t w0 = (uint32_t)p0 / S, w1 = (uint32_t)(p1 - 1) / S;
  if (w0 == w1) return;  // written by its wave
  auto at_of = [&](uint32_t w) __attribute__((always_inline)) {
    const int slot = w == w0 && (uint32_t)p0 != w0 * S ? 1 : 0;
    return ((int64_t)w * 2 + slot) * a.group + h;
  };
  float M = -INFINITY;
  for (uint32_t w = w0; w <= w1; ++w) M = fmaxf(M, ld_const(a.ml + at_of(w) * 2));
  float O = 0.f, L = 0.f;
  for (uint32_t w = w0; w <= w1; ++w) {
    const int64_t at = at_of(w);
    const float m = ld_const(a.ml + at * 2);
    const float f = m == -INFINITY ? 0.f : exp2_fast(m - M);
    O += f * a.part[at * kHeadDim + tid];
    L += f * ld_const(a.ml + at * 2 + 1);
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
  const size_t lds = (size_t)(2 * pairs + 1) * 4;
  hipLaunchKernelGGL(attn_fp4_span_kernel, dim3((unsigned)(device_cus() * kWgsPerCu)),
                     dim3(kThreads4), lds, st, a);
  hipLaunchKernelGGL(attn_fp4_merge_kernel, dim3((unsigned)(pairs * group)), dim3(kHeadDim), 0, st,
                     a);
  return check_launch(fn);
}
