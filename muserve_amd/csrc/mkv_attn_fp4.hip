// mkv_attn_fp4.hip — paged decode attention over a 4-bit pool (gfx950): rows of
// e2m1 codes and e8m0 scales (mkv_quant.h), dequantised in registers.
//
// One query token per sequence attends to the first seq_lens[b] cached tokens
// of its block table: softmax(q k^T * scale) v for each of the G query heads
// that share a KV head. A cached token and head is 2 x 136 bytes for 1024 * G
// flop, so HBM bounds the launch where there is much to read, and the chain of
// a span's first loads (1.2 us to the sequence, 2.8 to its K), its end (1.6)
// and the second kernel (4) where there is little. Measured: 256 sequences, 4
// query heads on a KV head, 439 MB, 76-83 us and 5 us for the second kernel; 2
// sequences of 131072 tokens, 16 on 2, 143 MB, 35 and 6 us; 1 sequence of 2000
// tokens, 4 on 1, 7 and 3 us.
//   * Work split: the sequences' tiles of 32 tokens (two pages) form one flat
//     list, with one place more for each sequence, about what its start and end
//     cost. Each wave of the resident grid takes a contiguous span of it, for
//     one KV head; a span's KV heads are neighbouring workgroups of one XCD,
//     which read the same lines of the rows at about the same time. Pieces of
//     sequences that spans cut leave (max, sum, unnormalised output) for a
//     second kernel to join; where a workgroup's four spans lie in one sequence
//     they leave one piece. (Spans by workgroup, its waves taking the tiles in
//     turn: a barrier for each sequence, 87 us instead of 81 at batch 256.)
//     Short contexts take a workgroup for each (sequence, KV head) instead, and
//     no second kernel (by_pairs).
//   * Loads: page by page straight into a wave's LDS (global_load_lds, 16
//     bytes a lane), two tiles in flight, the page ids a tile ahead of them.
//     (Into registers in the operands' own order a K row is a line for every
//     lane: 90 us at batch 256; through registers to LDS: 97.)
//   * Scores on the matrix cores (16x16x32 bf16): A = the 16 K rows of a page,
//     codes converted to bf16 with their scale (exact), B = the query heads in
//     columns n and n + 8. A column's lanes hold 8 tokens each; the maximum is
//     lazy (raised when a score passes it by 2^8), so most tiles need no
//     reduction over lanes, and each lane sums its own tokens' weights.
//   * P V on the matrix cores: A = the weights in two bf16 parts (the rows n
//     hold the weight rounded, the rows n + 8 what that left, rounded: within
//     2^-18 of the weight, to either side, for the price of rows that would be
//     empty), B = V, 16 dims a lane. The score tile's lanes already hold the A
//     operand: the tokens' order inside the product is free, so V is read in
//     theirs.
#include <math.h>

#include <atomic>

#include "mkv_dma.h"
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
// A row in LDS: the nine aligned 16-byte chunks that it lies in (a row starts at a
// multiple of 8, at byte 0 or 8 of its first chunk; an odd row's last chunk ends with it, an
// even row has one behind it). Eight rows lie on different banks.
constexpr int kRowLds = 144;
constexpr int kPage = 16 * kRowLds;  // bytes of a page of one head there
constexpr int kTileLds = 4 * kPage;  // a tile: K's two pages, then V's
constexpr int kPageLoads = (kPage + 1023) / 1024;  // instructions of a page
constexpr int kMaxGroup = 8;         // query heads per KV head
constexpr int kMaxPairs = 4096;      // batch x KV heads
constexpr int kXcds = 8;             // MI355X: workgroups go round robin over 8 XCDs
constexpr int kWgsPerCu = 2;
constexpr int kPairWaves = 8;        // of a workgroup that takes a whole (sequence, KV head)
constexpr int kPairTiles = 24;       // tiles of the longest sequence up to which they do, and
constexpr int kPairMore = 16;        // as many more with a sequence for each CU
constexpr int kWideSpans = 256;      // spans of a sequence from which the merge takes 16 waves
constexpr float kRaise = 8.f;        // log2 by which a score may pass the running maximum
// The maximum of a piece whose tokens' scores are all -inf: no weight beside any other
// piece, and told from the -inf of no tokens at all.
constexpr float kLowest = -3.402823466e38f;

struct Args {
  const uint8_t* q;      // [B, Hkv * G, 256] bf16
  const uint8_t* k;      // [P, 16, Hkv, 136]
  const uint8_t* v;
  const int32_t* table;  // [B, tstride]
  const int32_t* lens;   // [B]
  uint8_t* out;          // [B, Hkv * G, 256] bf16
  int32_t* hdr;          // workspace: the spans' sizes
  int32_t* pre;          // [B + 1] each sequence's first place
  float* ml;             // [spans, Hkv, 2, G, 2] (max, sum) of cut pieces, log2 units
  float* part;           // [spans, Hkv, 2, G, 256] their unnormalised outputs
  int64_t num_pages, tstride, shared_below;
  int32_t twidth, hkv, group, max_len, batch;
  float scale_log2;
  int32_t* err;
};

// The spans of the flat list: `least` places each, the first `more` one more.
struct Spans {
  int32_t least, more;
  __device__ __forceinline__ int32_t start(int32_t u) const {
    return u * least + (u < more ? u : more);
  }
  __device__ __forceinline__ int32_t of(int32_t place) const {  // of a place of the list
    const int32_t head = more * (least + 1);
    return place < head ? place / (least + 1) : more + (place - head) / least;
  }
  // whether the workgroup with span `first` has all its spans, and in the places p0 .. p1
  __device__ __forceinline__ bool whole(int32_t first, int32_t p0, int32_t p1) const {
    const int32_t s = start(first), e = start(first + kWaves);
    return e - s >= kWaves && s >= p0 && e <= p1;
  }
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ T lds_get(uint32_t at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) T*>(at);
}
// The places of a sequence in the flat list.
__device__ __forceinline__ int32_t places_of(int32_t len) {
  return len > 0 ? (len + kTile - 1) / kTile + 1 : 0;
}
// An output of the weights' sum L and the maximum M: the quotient; zeros of no tokens; NaN
// where there were some and all their scores were -inf (M is kLowest then, not -inf).
__device__ __forceinline__ float inverse_of(float L, float M) {
  return L == 0.f && M == -INFINITY ? 0.f : 1.f / L;  // (0 * inf: NaN)
}
// Eight codes of a word times the scale, as eight bf16.
__device__ __forceinline__ u32x4 dequant8(uint32_t w, float s) {
  return u32x4{mkv_fp4_pair(w, 0, s), mkv_fp4_pair(w, 1, s), mkv_fp4_pair(w, 2, s),
               mkv_fp4_pair(w, 3, s)};
}

// PAIR: a workgroup a (sequence, KV head), its waves taking the tiles in turn and joining
// their pieces in LDS: no second kernel, no prefix over the sequences.
template <bool PAIR>
__global__ __launch_bounds__(PAIR ? 64 * kPairWaves : kThreads4, 2) void attn_fp4_kernel(Args a) {
  constexpr int WAVES = PAIR ? kPairWaves : kWaves, STEP = PAIR ? WAVES : 1;
  // two tiles for each wave (in the end its piece [G][256]), the pieces' (m, l) [waves][G][2]
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t hkv = a.hkv;
  const int64_t cap = (int64_t)a.twidth * 16 < a.max_len ? (int64_t)a.twidth * 16 : a.max_len;
  // a sequence's cached tokens, cut to the table and the launch's bound
  auto length_of = [&](int b) __attribute__((always_inline)) {
    const int64_t len = ld_const(a.lens + b);
    return (int32_t)(len < 0 ? 0 : (len > cap ? cap : len));
  };
  // a sequence as the walk over the span has it: its tiles' places are pre0 .. pre1
  struct Seq {
    int32_t b, pre0, pre1, len;
  };
  auto next_seq = [&](Seq x) __attribute__((always_inline)) {  // the next one with tiles
    do {
      ++x.b;
      x.len = __builtin_amdgcn_readfirstlane(length_of(x.b));
    } while (x.len == 0);
    x.pre0 = x.pre1 + 1;
    x.pre1 = x.pre0 + (x.len + kTile - 1) / kTile;
    return x;
  };
  Seq cur;             // the sequence that is worked on
  Spans cut;
  int32_t head;        // KV head
  int32_t first, span;  // the workgroup's first span and the wave's: the places s0 .. s1
  int32_t s0, s1, fa;  // fa: the wave's next tile whose page ids are read
  if constexpr (PAIR) {
    const int32_t b = blockIdx.x / hkv;
    head = blockIdx.x - b * hkv;
    const int64_t given = ld_const(a.lens + b);
    if ((given > cap || given < 0) && head == 0 && tid == 0) raise_err(a.err, MKV_DEVERR_TABLE);
    cur.b = b;
    cur.pre0 = s0 = 0;
    cur.len = length_of(b);
    cur.pre1 = s1 = (cur.len + kTile - 1) / kTile;
    if (s1 == 0) {
      if (tid < a.group * 32)
        st16(a.out + ((int64_t)blockIdx.x * a.group * 32 + tid) * 16, u32x4{0u, 0u, 0u, 0u});
      return;
    }
    fa = wave;
  } else {
    __shared__ int32_t wave_tot[kWaves];
    __shared__ int32_t start_l[kWaves][2];  // (sequence, its first tile) that a span starts in
    // exclusive prefix of the places of 256 sequences from `base` on (a place for each
    // tile and one more), behind `before`; the round's total goes to `round`
    auto scan = [&](int base, int32_t before, int32_t& cnt, int32_t& round)
        __attribute__((always_inline)) {
      const int b = base + tid;
      cnt = b < a.batch ? places_of(length_of(b)) : 0;
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
    for (int base = 0; base < a.batch; base += kThreads4) {
      at = scan(base, T, cnt, round);
      T += round;
    }
    // Workgroups of one XCD (those with the same number modulo 8) take neighbouring spans.
    const int32_t xcd = blockIdx.x % kXcds, all = gridDim.x;
    const int32_t unit = xcd * (all / kXcds) + (xcd < all % kXcds ? xcd : all % kXcds) +
                         (int32_t)blockIdx.x / kXcds;
    head = unit % hkv;
    const int32_t total = T;
    T = T > 0 ? T - 1 : 0;  // (nothing starts at the place behind the last sequence)
    const int32_t spans = all / hkv * kWaves;
    cut = {T / spans, T % spans};
    first = unit / hkv * kWaves;
    span = first + wave;
    // The sequences that this workgroup's spans start in (and, by workgroup 0, the prefixes
    // for the merge kernel); a round's prefix is still held where there is one round.
    {
      int32_t before = 0;
      for (int base = 0; base < a.batch; base += kThreads4) {
        if (a.batch > kThreads4) {
          at = scan(base, before, cnt, round);
          before += round;
        }
        const int b = base + tid;
        if (b < a.batch) {
#pragma unroll
          for (int w = 0; w < kWaves; ++w) {
            const int32_t s = cut.start(first + w);
            if (s >= at && s < at + cnt) {
              start_l[w][0] = b;
              start_l[w][1] = at;
            }
          }
          if (blockIdx.x == 0) {
            a.pre[b] = at;
            const int64_t len = ld_const(a.lens + b);
            if (len > cap || len < 0) raise_err(a.err, MKV_DEVERR_TABLE);
          }
        }
      }
      if (blockIdx.x == 0 && tid == 0) {
        a.pre[a.batch] = total;
        a.hdr[0] = cut.least;
        a.hdr[1] = cut.more;
      }
      __syncthreads();
    }
    s0 = cut.start(span);
    s1 = cut.start(span + 1);
    if (s0 >= s1) return;  // (no barrier follows, but for workgroups with four spans)
    cur.b = __builtin_amdgcn_readfirstlane(start_l[wave][0]);
    cur.pre0 = __builtin_amdgcn_readfirstlane(start_l[wave][1]);
    cur.len = __builtin_amdgcn_readfirstlane(length_of(cur.b));
    cur.pre1 = cur.pre0 + (cur.len + kTile - 1) / kTile;
    fa = s0;
    if (fa == cur.pre1) {  // the span starts at the place behind a sequence
      if (++fa == s1) return;
      cur = next_seq(cur);
    }
  }

  // Of the two waves on a SIMD the arbiter favours the older one: with it alone the first
  // workgroup of a CU ends a third before the second. They take turns, tile by tile.
  const uint32_t wslot = __builtin_amdgcn_s_getreg((3 << 11) | 4) & 1u;
  const int c = lane & 15, g = lane >> 4;  // row / column and quad of a matrix operand
  const uint32_t rest_mask = c < 8 ? 0u : ~0u;  // the lane takes a weight's first part off
  const int32_t row_bytes = hkv * kFp4Row;
  // page ids read through the caches: shared ones, and all where KV heads share lines
  const int64_t hot_below = hkv > 1 ? a.num_pages : a.shared_below;
  const uint32_t num_pages = a.num_pages < INT32_MAX ? (uint32_t)a.num_pages : INT32_MAX;
  float* ml_l = reinterpret_cast<float*>(lds + 2 * WAVES * kTileLds);
  const uint32_t tile_l = lds_addr(lds + wave * 2 * kTileLds);
  const uint32_t odd_k = ((c * hkv + head) & 1) * 8;  // where a row starts in its first chunk
  const uint32_t odd_v[2] = {(head & 1) * 8u, ((hkv + head) & 1) * 8u};  // of rows 4 g + j, j even, odd
  const uint32_t get_k = c * kRowLds + odd_k + 16 * g;  // dims 32 g .. and 128 + 32 g ..
  const uint32_t get_ks = c * kRowLds + odd_k + kFp4Codes + g;
  const uint32_t get_v = 2 * kPage + 4 * g * kRowLds + 8 * c;  // dims 16 c ..
  const uint32_t get_vs = 2 * kPage + 4 * g * kRowLds + kFp4Codes + c / 2;
  uint32_t chunk_off[kPageLoads];  // of a page's rows of this head, chunk 64 j + lane
#pragma unroll
  for (int j = 0; j < kPageLoads; ++j) {
    const int i = 64 * j + lane, r = i / (kRowLds / 16);
    chunk_off[j] = ((r * row_bytes + head * kFp4Row) & ~15) + 16 * (i % (kRowLds / 16));
  }

  Seq ahead = cur;  // of the tile whose page ids are read next

  // The pages of a tile. Their ids are read a tile ahead of the rows' loads, which wait for
  // them; a tile's K and V are loaded once the tile two before it has been read.
  struct Pages {
    int32_t id0, id1, left;  // left: the tile's tokens and those behind it, 0: no tile
  };
  auto read_ids = [&]() __attribute__((always_inline)) {
    Pages x = {0, 0, 0};
    if (!PAIR && fa == ahead.pre1 && ++fa < s1) ahead = next_seq(ahead);
    if (fa < s1) {
      const int32_t tok0 = (fa - ahead.pre0) * kTile;
      const int32_t* ids = a.table + (int64_t)ahead.b * a.tstride + tok0 / 16;
      x.left = ahead.len - tok0;
      x.id0 = ld_const(ids);
      x.id1 = ld_const(ids + (x.left > 16 ? 1 : 0));
      fa += STEP;
    }
    return x;
  };
  struct Where {
    int64_t base0, base1;    // of the pages' rows in both planes
    int32_t valid0, valid1;  // tokens of the two pages
    int32_t hot;             // bit i: page i is read through the caches
    bool there;              // there is such a tile
  };
  auto locate = [&](Pages x) __attribute__((always_inline)) {
    Where w;
    w.hot = 0;
    w.there = x.left > 0;
    auto page = [&](int i, int32_t id, int32_t left, int64_t& base, int32_t& valid)
        __attribute__((always_inline)) {
      valid = left < 0 ? 0 : (left > 16 ? 16 : left);
      if ((uint32_t)id >= num_pages) {  // no token of a page id outside the pool
        if (lane == 0 && left > 0) raise_err(a.err, MKV_DEVERR_PAGE);
        id = 0;
        valid = 0;
      }
      w.hot |= id < hot_below ? 1 << i : 0;
      base = (int64_t)id * (16 * row_bytes);
    };
    page(0, x.id0, x.left, w.base0, w.valid0);
    page(1, x.id1, x.left - 16, w.base1, w.valid1);
    return w;
  };
  // a page's rows to LDS, kPageLoads instructions
  auto load_page = [&](const uint8_t* src, uint32_t dst, bool hot) __attribute__((always_inline)) {
    lds_reads_done();
    constexpr int kRest = (kPage % 1024) / 16;  // chunks of the last instruction
    if (hot) {
      dma16_cached(src, chunk_off[0], dst);
      dma16_cached(src, chunk_off[1], dst + 1024);
      if (lane < kRest) dma16_cached(src, chunk_off[2], dst + 2048);
    } else {
      dma16(src, chunk_off[0], dst);
      dma16(src, chunk_off[1], dst + 1024);
      if (lane < kRest) dma16(src, chunk_off[2], dst + 2048);
    }
  };
  auto load_k = [&](Where w, uint32_t slot) __attribute__((always_inline)) {
    load_page(a.k + w.base0, slot, w.hot & 1);
    load_page(a.k + w.base1, slot + kPage, w.hot & 2);
  };
  auto load_v = [&](Where w, uint32_t slot) __attribute__((always_inline)) {
    load_page(a.v + w.base0, slot + 2 * kPage, w.hot & 1);
    load_page(a.v + w.base1, slot + 3 * kPage, w.hot & 2);
  };

  u32x4 qb[8];
  f32x4 acc[16];
  float m_run, l_run;
  int32_t f = fa;          // the place of the tile that is computed next
  uint32_t slot = tile_l;  // and where it lies
  const uint32_t both = 2 * tile_l + kTileLds;
  Where now = locate(read_ids());
  if (!PAIR || now.there) {
    load_k(now, slot);
    load_v(now, slot);
  }
  Where next = locate(read_ids());
  if (next.there) {
    load_k(next, both - slot);
    load_v(next, both - slot);
  }
  Pages pages = read_ids();
  auto load_q = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 8; ++s) {  // the dims of K's operand: 32 g + 8 s, 128 + 32 g + 8 (s - 4)
      // (columns behind the last head repeat it: their results are not used)
      const int h = (c & 7) < a.group ? (c & 7) : a.group - 1;
      const int dim = 32 * g + 8 * (s & 3) + 128 * (s >> 2);
      qb[s] = ld16(a.q + (((int64_t)cur.b * hkv + head) * a.group + h) * kQRow + 2 * dim);
    }
  };
  load_q();
  for (;;) {  // the span's sequences
    const int32_t end = cur.pre1 < s1 ? cur.pre1 : s1;
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run = -INFINITY;
    l_run = 0.f;
    bool some = false;  // a token of the sequence in a page of the pool
    while (f < end) {
      __builtin_amdgcn_s_setprio(0);
      if (((uint32_t)(f / STEP + wslot) & 1u) != 0) __builtin_amdgcn_s_setprio(1);
      const bool has1 = next.there;
      // the tile's K has come once what was asked for behind it is all that is in flight
      if (has1) vm_wait_n<6 * kPageLoads>(); else vm_wait_n<2 * kPageLoads>();
      u32x4 k[2][2];
      float ks[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          k[i][h] = lds_get<u32x4a8>(slot + i * kPage + get_k + 64 * h);
          ks[i][h] = fp4_scale(lds_get<uint8_t>(slot + i * kPage + get_ks + 4 * h));
        }
      const Where after = locate(pages);
      const bool has2 = after.there;
      if (has2) load_k(after, slot);
      pages = read_ids();
      // scores: lane (c, g) gets tokens 4 g + j of each page, for head c & 7
      float sv[8];
      {
        f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            sc[i] = mfma(dequant8(k[i][s >> 2][s & 3], ks[i][s >> 2]), qb[s], sc[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) sv[j] = sc[j >> 2][j & 3] * a.scale_log2;
      }
      const bool part = now.valid0 < 16 || now.valid1 < 16;
      some |= now.valid0 + now.valid1 > 0;
      if (part) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          sv[j] = 4 * g + (j & 3) < (j < 4 ? now.valid0 : now.valid1) ? sv[j] : -INFINITY;
      }
      const float mx = fmaxf(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])),
                             fmaxf(fmaxf(sv[4], sv[5]), fmaxf(sv[6], sv[7])));
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
        // the weight's bf16 in rows below 8, in the others that of what it left (exact)
        const uint32_t near = pack_bf16(p0, p1) & rest_mask;
        pa[j / 2] = pack_bf16(p0 - bits_f32(near << 16), p1 - bits_f32(near & 0xffff0000u));
      }
      if (has2) vm_wait_n<6 * kPageLoads>();
      else if (has1) vm_wait_n<4 * kPageLoads>();
      else vm_wait_n<0>();
      u32x2 v[8];
      float vsc[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t row = (j >> 2) * kPage + (j & 3) * kRowLds + odd_v[j & 1];
        v[j] = lds_get<u32x2>(slot + get_v + row);
        vsc[j] = fp4_scale(lds_get<uint8_t>(slot + get_vs + row));
      }
      if (has2) load_v(after, slot);
      if (part) {  // rows that hold anything: zeros
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool ok = 4 * g + (j & 3) < (j < 4 ? now.valid0 : now.valid1);
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
      now = next;
      next = after;
      slot = both - slot;
      f += STEP;
    }
    const Seq done = cur;
    const bool last = PAIR || cur.pre1 + 1 >= s1;
    if (!last) {  // the next sequence's query rows come while this one's piece goes
      cur = next_seq(cur);
      f = cur.pre0;
      load_q();
    }
    // The sequence's piece in this span: the quads' sums, and those of the weights' two
    // parts, which the wave's halves hold. A swap of the halves of two tiles leaves both sums
    // in half the registers: lanes below 32 have the dims 16 c .. + 7, the others 16 c + 8 ..,
    // of the heads 4 (g % 2) + i.
    const float l = over_rows<4>(l_run, [](float x, float y) { return x + y; });
    const float m_end = m_run == -INFINITY && some ? kLowest : m_run;
    float o[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(f32_bits(acc[j][i]), f32_bits(acc[j + 8][i]),
                                                        false, false);
        o[j][i] = bits_f32(r[0]) + bits_f32(r[1]);
      }
    const int h0 = 4 * (g & 1), d0 = 16 * c + 8 * (g >> 1);
    uint8_t* out = a.out + ((int64_t)done.b * hkv + head) * a.group * kQRow;
    // the workgroup's spans lie in one sequence: one piece, its first span's
    const bool joint = PAIR || cut.whole(first, done.pre0, done.pre1);
    const bool whole = !PAIR && done.pre0 >= s0 && done.pre1 <= s1;
    // (cut sequences: the span's first goes to slot 0, its last to slot 1)
    const int64_t piece =
        PAIR ? 0 : (((int64_t)span * hkv + head) * 2 + (done.pre0 <= s0 ? 0 : 1)) * a.group;
    float* piece_l = reinterpret_cast<float*>(lds + wave * 2 * kTileLds);
    if (lane < a.group) {
      float* ml = joint ? ml_l + (wave * a.group + lane) * 2 : a.ml + (piece + lane) * 2;
      if (!whole) {
        ml[0] = m_end;
        ml[1] = l;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = h0 + i;
      const float inv = __shfl(inverse_of(l, m_end), h);
      if (h >= a.group) continue;
      if (whole) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack_bf16(o[2 * j][i] * inv, o[2 * j + 1][i] * inv);
        st16(out + h * kQRow + 2 * d0, u32x4{w[0], w[1], w[2], w[3]});
      } else {
        float* dst = (joint ? piece_l + h * kHeadDim : a.part + (piece + h) * kHeadDim) + d0;
        *reinterpret_cast<f32x4*>(dst) = f32x4{o[0][i], o[1][i], o[2][i], o[3][i]};
        *reinterpret_cast<f32x4*>(dst + 4) = f32x4{o[4][i], o[5][i], o[6][i], o[7][i]};
      }
    }
    if (joint) {
      __syncthreads();
      const int64_t at = PAIR ? 0 : ((int64_t)first * hkv + head) * 2 * a.group;
      for (int h = wave; h < a.group; h += WAVES) {  // a head a wave, four dims a lane
        float m[WAVES], ls[WAVES], M = -INFINITY, L = 0.f;
        f32x4 x[WAVES], O = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          m[w] = ml_l[(w * a.group + h) * 2];
          ls[w] = ml_l[(w * a.group + h) * 2 + 1];
          x[w] = reinterpret_cast<const f32x4*>(lds + w * 2 * kTileLds)[h * (kHeadDim / 4) + lane];
        }
#pragma unroll
        for (int w = 0; w < WAVES; ++w) M = fmaxf(M, m[w]);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          // (a wave without a score: 1, so that a NaN of its sums stays)
          const float e = m[w] == -INFINITY ? 1.f : exp2_fast(m[w] - M);
#pragma unroll
          for (int d = 0; d < 4; ++d) O[d] += e * x[w][d];
          L += e * ls[w];
        }
        if constexpr (PAIR) {
          const float inv = inverse_of(L, M);
          *reinterpret_cast<u32x2*>(out + h * kQRow + 8 * lane) =
              u32x2{pack_bf16(O[0] * inv, O[1] * inv), pack_bf16(O[2] * inv, O[3] * inv)};
        } else {
          *reinterpret_cast<f32x4*>(a.part + (at + h) * kHeadDim + 4 * lane) = O;
          if (lane == 0) {
            a.ml[(at + h) * 2] = M;
            a.ml[(at + h) * 2 + 1] = L;
          }
        }
      }
    }
    if (last) return;
  }
}

// Joins the pieces of one (pair, query head) that spans cut, and writes the zeros of an
// empty pair. Wave w takes the pieces w, w + WAVES, .., four dims a lane, BATCH of them
// in flight; the waves' sums are joined in LDS. WAVES is 16 where a sequence lies in many
// spans, else 4. Measured (us of both kernels with 4 waves and with 16; a sequence's spans,
// and the pieces that workgroups whose spans all lie in it leave of them): 1 sequence of 4096
// tokens (128 spans, 32 pieces) 10.8, 11.7, of 32768 (1024, 256) 21.8, 17.4; 8 of 4096 (128,
// 32) 13.7, 13.9, of 32768 (256, 66) 25.0, 24.0; 2 of 100000 and two KV heads (512, 128) 34.4,
// 32.2; 128 of 4096 (16, 6 to 8) 33.8, 35.6.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attn_fp4_merge_kernel(Args a) {
  constexpr int BATCH = 8;
  __shared__ __attribute__((aligned(16))) float wave_o[WAVES][kHeadDim];
  __shared__ float wave_ml[WAVES][2];
  const int pr = blockIdx.x / a.group, h = blockIdx.x % a.group;
  const int b = pr / a.hkv, head = pr - b * a.hkv;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Spans cut = {ld_const(a.hdr), ld_const(a.hdr + 1)};  // (with the sequence's bounds)
  const int32_t p0 = ld_const(a.pre + b);
  int32_t p1 = ld_const(a.pre + b + 1);
  asm volatile("" ::"s"(cut.least), "s"(cut.more));
  uint16_t* out = reinterpret_cast<uint16_t*>(a.out + ((int64_t)pr * a.group + h) * kQRow);
  if (p1 <= p0) {
    if (tid < kHeadDim) out[tid] = 0;
    return;
  }
  --p1;  // without the place behind its tiles
  const int32_t u0 = cut.of(p0), u1 = cut.of(p1 - 1);
  if (u0 == u1) return;  // written with its span
  // spans u0 .. u1; those of the workgroups g0 .. g1 that lie in the sequence as one each
  int32_t g0 = u0 / kWaves, g1 = u1 / kWaves + 1;
  g0 += cut.start(g0 * kWaves) < p0 ? 1 : 0;
  g1 -= cut.whole(kWaves * (g1 - 1), p0, p1) ? 0 : 1;
  const int mid = g1 > g0 ? g1 - g0 : 0;
  const int lead = mid > 0 ? kWaves * g0 - u0 : u1 - u0 + 1;
  const int n = lead + mid + (mid > 0 ? u1 + 1 - kWaves * g1 : 0);
  auto at_of = [&](int i) __attribute__((always_inline)) {
    const int32_t u = i < lead ? u0 + i
                               : (i < lead + mid ? kWaves * (g0 + i - lead)
                                                 : kWaves * g1 + (i - lead - mid));
    const int slot = u == u0 && p0 != cut.start(u0) ? 1 : 0;
    return (((int64_t)u * a.hkv + head) * 2 + slot) * a.group + h;
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
  out[tid] = f32_to_bf16_rne(L == 0.f ? O * inverse_of(L, M) : O / L);
}

// Workgroups of spans: the resident ones, as many for each KV head.
int64_t span_grid(int32_t hkv) {
  const int64_t fit = (int64_t)device_cus() * kWgsPerCu / hkv;
  return (fit < 1 ? 1 : fit) * hkv;
}
// Whether each (sequence, KV head) gets a workgroup: for short contexts, where that costs
// less than the prefix and the second kernel do. Measured (us by spans and by pairs, 4
// query heads): 1 sequence of 512 tokens 9.9, 8.8, of 1024 10.2, 12.6; 64 of 1024 14.3,
// 14.6, of 2048 18.5, 23.3; 256 of 512 20.2, 11.1, of 1024 25.7, 16.7, lognormal up to 1024
// 18.6, 15.0, up to 2048 23.5, 23.7; 512 of 1024 40.5, 33.8, lognormal 28.2, 27.1.
bool by_pairs(int64_t pairs, int64_t max_len) {
  const int64_t cus = device_cus();
  if (pairs > 2 * cus) return false;
  const int64_t some = pairs < cus ? pairs : cus;
  return max_len <= (kPairTiles + kPairMore * some / cus) * kTile;
}

struct WsLayout {
  int64_t pre, ml, part, total;
};
WsLayout ws_layout(int64_t batch, int32_t hkv, int64_t group, int64_t max_len) {
  if (by_pairs(batch * hkv, max_len)) return WsLayout{0, 0, 0, 0};
  const int64_t pieces = span_grid(hkv) * kWaves * 2 * group;
  WsLayout w;
  w.pre = 256;
  w.ml = w.pre + ((batch + 1) * 4 + 255) / 256 * 256;
  w.part = w.ml + (pieces * 2 * 4 + 255) / 256 * 256;
  w.total = w.part + pieces * kHeadDim * 4;
  return w;
}

// Launches `grid` workgroups, once their LDS has been asked for on this device.
template <bool PAIR>
int launch(const Args& a, int64_t grid, hipStream_t st, const char* fn) {
  constexpr int WAVES = PAIR ? kPairWaves : kWaves;
  constexpr size_t most = WAVES * (2 * kTileLds + kMaxGroup * 2 * 4);
  static std::atomic<uint64_t> asked[16];  // a bit a device
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  const uint64_t bit = 1ull << (dev & 63);
  std::atomic<uint64_t>& word = asked[(dev >> 6) & 15];
  if (!(word.load(std::memory_order_relaxed) & bit)) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(attn_fp4_kernel<PAIR>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, most) != hipSuccess)
      return set_error(MKV_E_LAUNCH, "%s: %zu bytes of LDS refused", fn, most);
    word.fetch_or(bit, std::memory_order_relaxed);
  }
  const size_t lds = WAVES * (2 * kTileLds + (size_t)a.group * 2 * 4);
  hipLaunchKernelGGL(attn_fp4_kernel<PAIR>, dim3((unsigned)grid), dim3(64 * WAVES), lds, st, a);
  return MKV_OK;
}

bool shape_ok(int32_t batch, int32_t hkv, int32_t hq) {
  if (batch < 0 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || hq / hkv > kMaxGroup) return false;
  return (int64_t)batch * hkv <= kMaxPairs;
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" int64_t mkv_decode_attention_fp4_workspace_bytes(int32_t batch, int32_t num_kv_heads,
                                                            int32_t num_q_heads,
                                                            int32_t max_seq_len) {
  if (!shape_ok(batch, num_kv_heads, num_q_heads) || max_seq_len < 0) return -1;
  return ws_layout(batch, num_kv_heads, num_q_heads / num_kv_heads, max_seq_len).total;
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
  const WsLayout L = ws_layout(batch, num_kv_heads, group, max_seq_len);
  MKV_REQUIRE(L.total == 0 || (workspace && workspace_bytes >= L.total && aligned16(workspace)),
              MKV_E_INVALID,
              "%s: workspace of %lld bytes (16-byte aligned) required", fn, (long long)L.total);
  Args a;
  a.q = static_cast<const uint8_t*>(q);
  a.k = static_cast<const uint8_t*>(k_cache);
  a.v = static_cast<const uint8_t*>(v_cache);
  a.table = page_table;
  a.lens = seq_lens;
  a.out = static_cast<uint8_t*>(out);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.hdr = reinterpret_cast<int32_t*>(ws);
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
  a.batch = batch;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.err = err;
  const hipStream_t st = as_stream(stream);
  if (L.total == 0) {
    const int rc = launch<true>(a, pairs, st, fn);
    return rc != MKV_OK ? rc : check_launch(fn);
  }
  const int rc = launch<false>(a, span_grid(num_kv_heads), st, fn);
  if (rc != MKV_OK) return rc;
  // spans of a sequence: about its share of them, and at most one for each of its tiles
  const int64_t tiles = ((int64_t)max_seq_len + kTile - 1) / kTile;
  const int64_t spans = span_grid(num_kv_heads) / num_kv_heads * kWaves / batch;
  if (tiles >= kWideSpans && spans >= kWideSpans)
    hipLaunchKernelGGL(attn_fp4_merge_kernel<16>, dim3((unsigned)(pairs * group)), dim3(16 * 64), 0,
                       st, a);
  else
    hipLaunchKernelGGL(attn_fp4_merge_kernel<4>, dim3((unsigned)(pairs * group)), dim3(4 * 64), 0,
                       st, a);
  return check_launch(fn);
}
