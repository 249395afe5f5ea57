// mkv_fp4.hip — bf16 -> 4-bit quantize-on-append and 4-bit -> bf16 gather for
// gfx950 (rows of e2m1 codes and e8m0 scales: mkv_quant.h).
#include "mkv_quant.h"

namespace mkv {
namespace {

constexpr int kHeadDim = 256;
constexpr int kLanesPerRow = 16;                     // 16 values a lane, two lanes a block
constexpr int kRowsPerWg = kThreads / kLanesPerRow;  // 16

struct AppendFp4Args {
  uint8_t* k_pool;
  uint8_t* v_pool;
  int64_t pool_layer_stride;
  int64_t num_slots;
  const uint8_t* k_src;
  const uint8_t* v_src;
  int64_t src_layer_stride;
  int64_t src_token_stride;
  const int64_t* slots;
  uint32_t num_rows;  // tokens * heads
  uint32_t num_heads;
  int32_t* err;
};

// One 16-lane group per (token, head) row of one (layer, K|V): grid.x covers the
// rows, grid.y is layer * 2 + K|V. HEADS is the head count when it is 1 or 2 (0: any),
// which saves the division by it (us a call in a graph, known and by division: one head, 77
// tokens 2.07, 2.09, 1000 2.13, 2.17, 4096 2.40, 2.44; two heads, 4096 3.80, 3.88; from
// 16384 tokens on the same).
// 512 bytes in and 136 out for a row: HBM bounds a long one, a chunk of a few thousand
// tokens is little more than its launch (77 tokens 2.5 us, 999 of two heads 3.0, 16384
// 6-7 us: 3.0-3.5 TB/s).
template <int HEADS>
__global__ __launch_bounds__(kThreads) void append_fp4_kernel(AppendFp4Args a) {
  const uint32_t lane = threadIdx.x & (kLanesPerRow - 1);
  const uint32_t row = blockIdx.x * kRowsPerWg + threadIdx.x / kLanesPerRow;
  if (row >= a.num_rows) return;
  const uint32_t l = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1u;
  const uint32_t nh = HEADS ? (uint32_t)HEADS : a.num_heads;
  const uint32_t t = row / nh;
  const uint32_t h = row - t * nh;
  const int64_t slot = a.slots[t];
  const uint8_t* src = (is_v ? a.v_src : a.k_src) + (int64_t)l * a.src_layer_stride +
                       (int64_t)t * a.src_token_stride + (int64_t)h * (kHeadDim * 2) + lane * 32;
  const u32x4 r0 = ld_nt(src), r1 = ld_nt(src + 16);
  if (slot < 0 || slot >= a.num_slots) {  // -1 skips the token; anything else is an error
    if (slot != -1 && lane == 0 && h == 0 && !is_v) raise_err(a.err, MKV_DEVERR_SLOT);
    return;
  }
  const uint32_t w[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
  uint32_t c[2];
  const uint32_t byte = quantise_fp4<16>(w, c);
  uint8_t* dst = (is_v ? a.v_pool : a.k_pool) + (int64_t)l * a.pool_layer_stride +
                 (slot * nh + h) * kFp4Row;
  *reinterpret_cast<u32x2*>(dst + lane * 8) = u32x2{c[0], c[1]};
  if ((lane & 1) == 0) dst[kFp4Codes + lane / 2] = (uint8_t)byte;
}

// Gather: a tile is kGatherRows output rows of one (layer, K|V, sequence); 32 lanes take
// a (row, head): 8 codes and their block's scale byte in, 16 bytes out, a tile's rows
// loaded before the first is stored. 136 bytes in and 512 out for a row: HBM's writes
// bound it (65536 rows, 85 MB, 16.3 us: 5.2 TB/s). Tiles of 8 rows took 22.3 us, of 32
// 27.8, loads past the caches 22. The stores go through the caches: past them the gather
// alone takes 15.3 us, but the prefill attention that reads its window then finds less of
// it there (both together 453.5 us instead of 448.8).
constexpr int kGatherRows = 16;
constexpr int kGatherThreads = 256;

__global__ __launch_bounds__(kGatherThreads) void gather_fp4_kernel(GatherArgs a, int32_t heads) {
  constexpr int GROUPS = kGatherThreads / 32, EACH = kGatherRows / GROUPS;
  GatherTile<kGatherRows> t;
  t.init(a);
  const int64_t row_limit = a.out_offsets ? t.nvalid : a.out_len;
  if (t.row0 >= row_limit) return;
  t.locate(a);
  t.load_pages(a);
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
  const uint8_t* plane = (t.is_v ? a.v_pool : a.k_pool) + (int64_t)t.layer * a.pool_layer_stride;
  uint8_t* out = (t.is_v ? a.v_out : a.k_out) + (int64_t)t.layer * a.out_layer_stride;
  const uint8_t* src[EACH];  // null: a row past the data, or of a bad page id
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int r = e * GROUPS + group;
    const int64_t p = t.p0 + r;
    const int32_t page = t.row0 + r < t.nvalid ? t.page_of(p) : -1;
    src[e] = page < 0 ? nullptr : plane + ((int64_t)page * 16 + (p & 15)) * heads * kFp4Row;
  }
  for (int h = 0; h < heads; ++h) {
    uint32_t c[EACH], b[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      c[e] = b[e] = 0;
      if (src[e]) {
        c[e] = *reinterpret_cast<const uint32_t*>(src[e] + h * kFp4Row + lane * 4);
        b[e] = src[e][h * kFp4Row + kFp4Codes + lane / 4];
      }
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int r = e * GROUPS + group;
      const float s = fp4_scale(b[e]);
      if (t.row0 + r < row_limit)
        st16(out + ((t.out_row + r) * heads + h) * (kHeadDim * 2) + lane * 16,
             u32x4{mkv_fp4_pair(c[e], 0, s), mkv_fp4_pair(c[e], 1, s), mkv_fp4_pair(c[e], 2, s),
                   mkv_fp4_pair(c[e], 3, s)});
    }
  }
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" int mkv_append_fp4(void* k_pool, void* v_pool, int64_t pool_layer_stride,
                              int64_t num_slots, const void* k_src, const void* v_src,
                              int64_t src_layer_stride, int64_t src_token_stride,
                              const int64_t* slot_mapping, int64_t num_tokens, int32_t num_layers,
                              int32_t num_heads, int32_t head_dim, int32_t* err, void* stream) {
  clear_error();
  MKV_REQUIRE(num_tokens >= 0 && num_layers >= 0 && num_slots >= 0 && num_heads > 0,
              MKV_E_INVALID, "mkv_append_fp4: bad size");
  MKV_REQUIRE(head_dim == kHeadDim, MKV_E_UNSUPPORTED,
              "mkv_append_fp4: head_dim %d unsupported (only 256)", head_dim);
  if (num_tokens == 0 || num_layers == 0) return MKV_OK;
  MKV_REQUIRE(k_pool && v_pool && k_src && v_src && slot_mapping && err, MKV_E_INVALID,
              "mkv_append_fp4: null pointer");
  MKV_REQUIRE(aligned16(k_src) && aligned16(v_src) && src_layer_stride % 16 == 0 &&
                  src_token_stride % 16 == 0 && aligned16(k_pool) && aligned16(v_pool) &&
                  pool_layer_stride % 16 == 0,
              MKV_E_ALIGN, "mkv_append_fp4: misaligned pointer or stride");
  MKV_REQUIRE((uint64_t)num_tokens < (1ull << 31), MKV_E_UNSUPPORTED,
              "mkv_append_fp4: too many rows for one call");
  const uint64_t rows = (uint64_t)num_tokens * (uint64_t)num_heads;
  const int64_t wgs = (int64_t)((rows + kRowsPerWg - 1) / kRowsPerWg);
  MKV_REQUIRE(rows < (1ull << 31) && grid_fits(wgs, kThreads) && num_layers <= 32767,
              MKV_E_UNSUPPORTED, "mkv_append_fp4: too many rows for one call");
  AppendFp4Args a{(uint8_t*)k_pool, (uint8_t*)v_pool, pool_layer_stride, num_slots,
                  (const uint8_t*)k_src, (const uint8_t*)v_src, src_layer_stride,
                  src_token_stride, slot_mapping, (uint32_t)rows, (uint32_t)num_heads, err};
  dim3 grid((unsigned)wgs, (unsigned)(2 * num_layers));
  if (num_heads == 1)
    hipLaunchKernelGGL(append_fp4_kernel<1>, grid, dim3(kThreads), 0, as_stream(stream), a);
  else if (num_heads == 2)
    hipLaunchKernelGGL(append_fp4_kernel<2>, grid, dim3(kThreads), 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL(append_fp4_kernel<0>, grid, dim3(kThreads), 0, as_stream(stream), a);
  return check_launch("mkv_append_fp4");
}

extern "C" int mkv_gather_dequant_fp4(const void* k_pool, const void* v_pool,
                                      int64_t pool_layer_stride, int64_t num_pages,
                                      const int32_t* block_tables, int64_t table_stride,
                                      int32_t table_width, const int32_t* seq_lens,
                                      const int32_t* starts, int32_t batch, int64_t out_len,
                                      const int64_t* out_offsets, void* k_out, void* v_out,
                                      int64_t out_layer_stride, int32_t num_layers,
                                      int32_t num_heads, int32_t head_dim, int32_t* err,
                                      void* stream) {
  clear_error();
  MKV_REQUIRE(batch >= 0 && out_len >= 0 && num_layers >= 0 && num_pages >= 0 &&
                  table_width >= 0 && num_heads > 0,
              MKV_E_INVALID, "mkv_gather_dequant_fp4: bad size");
  MKV_REQUIRE(head_dim == kHeadDim && num_heads <= 1024, MKV_E_UNSUPPORTED,
              "mkv_gather_dequant_fp4: heads=%d head_dim=%d unsupported (up to 1024 heads of 256)",
              num_heads, head_dim);
  if (batch == 0 || out_len == 0 || num_layers == 0) return MKV_OK;
  MKV_REQUIRE(num_layers <= 32767, MKV_E_UNSUPPORTED,
              "mkv_gather_dequant_fp4: too many layers for one call");
  GatherArgs a;
  const int rc = fill_gather_args(a, "mkv_gather_dequant_fp4", k_pool, v_pool, pool_layer_stride,
                                  num_pages, block_tables, table_stride, table_width, seq_lens,
                                  starts, batch, out_len, out_offsets, k_out, v_out,
                                  out_layer_stride, num_heads * kHeadDim * 2, err);
  if (rc != MKV_OK) return rc;
  const dim3 grid = gather_grid(a, kGatherRows, num_layers);
  MKV_REQUIRE(grid_fits(grid.x, kGatherThreads), MKV_E_UNSUPPORTED,
              "mkv_gather_dequant_fp4: out_len too large");
  hipLaunchKernelGGL(gather_fp4_kernel, grid, dim3(kGatherThreads), 0, as_stream(stream), a,
                     num_heads);
  return check_launch("mkv_gather_dequant_fp4");
}
