// mkv_rope.hip — the RMS norm of each query and key head and the rotation by
// its position in one pass (gfx950), for the attention layer between its
// projections and the KV pool; K and V go straight into the pool where one is
// given (16-bit, fp8 or 4-bit pages), so K is neither written nor read twice.
//
// A row of head_dim values is one read and one write of 2 * head_dim bytes: HBM
// bounds a large launch (32768 tokens of 4 + 1 heads of 256, 168 MB, 29-33 us:
// 5.0-5.8 TB/s), and a small one is its launch and a chain of loads that wait for each
// other though none needs the one before: position, frequency, slot, weights (256
// tokens 4.1 us, with the append 4.2; 4096 tokens of a prefill chunk with the
// append 8.8, whose bytes would take 5.1 at a copy's rate). The pools' types, us a call
// in a graph of 16-bit, fp8 and 4-bit: 1 token 3.2, 3.7, 3.2; 256 tokens 3.5, 4.1, 3.5;
// 4096 8.4, 9.7, 8.5. head_dim / 8 lanes own a token and take its heads one after the
// other (16 bytes a lane), so a token's sines and cosines are computed once for
// all of its heads and stay in registers.
//
// Angles: position * inv_freq in fp64, reduced to a turn in fp64, so that far
// positions lose nothing; sine and cosine of the reduced angle in fp32. Norm, scale
// and rotation are fp32; the one rounding is to the output's type (fp8 and 4-bit
// pools quantise that rounded row, so the pool holds what appending K would).

#include "mkv_quant.h"

namespace mkv {
namespace {

constexpr int kRopeThreads = 256;

enum WeightKind { kNoWeight = 0, kWeightBf16 = 1, kWeightF16 = 2, kWeightF32 = 3 };
enum PoolKind { kPoolNone = 0, kPool16 = 1, kPoolFp8 = 2, kPoolFp4 = 3 };

struct RopeArgs {
  const uint8_t* src[3];                           // q, k, v
  int64_t token_stride[3], head_stride[3];         // bytes
  uint8_t* q_out;                                  // [tokens, hq, D]
  uint8_t* k_out;                                  // [tokens, hk, D] (no pool)
  uint8_t* pool[2];                                // K and V plane of one layer
  float* scale[2];                                 // fp8
  const int64_t* slots;
  int64_t num_slots;
  const int64_t* positions;
  const void* inv_freq;                            // [rot / 2] float or double
  const void* weight[2];                           // [D] of q and k, or null: no norm
  int64_t tokens;
  int32_t hq, hk, heads, per_wg;                   // all heads, heads of a workgroup
  int32_t rot, freq64, weight_kind;
  float eps, rope_scale, centre;                   // centre: 1 is added to the weights
  int32_t* err;
};

__device__ __forceinline__ float f16_lo(uint32_t w) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xffffu));
}
__device__ __forceinline__ float f16_hi(uint32_t w) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
}
template <bool F16>
__device__ __forceinline__ void unpack8(const u32x4 r, float (&x)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = F16 ? f16_lo(w[i]) : bf16_lo(w[i]);
    x[2 * i + 1] = F16 ? f16_hi(w[i]) : bf16_hi(w[i]);
  }
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (F16) {
    const uint16_t a = __builtin_bit_cast(uint16_t, (_Float16)lo);
    const uint16_t b = __builtin_bit_cast(uint16_t, (_Float16)hi);
    return a | (uint32_t)b << 16;
  } else {
    return pack_bf16(lo, hi);
  }
}
// Eight weights from dim d on, with the centre.
__device__ __forceinline__ void weights8(const void* w, int32_t kind, float centre, int d,
                                         float (&x)[8]) {
  if (kind == kWeightF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = reinterpret_cast<const float*>(w)[d + i];
  } else {
    const u32x4 r = ld16(reinterpret_cast<const uint8_t*>(w) + 2 * d);
    if (kind == kWeightBf16) unpack8<false>(r, x); else unpack8<true>(r, x);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] += centre;
}

template <int D, bool F16, bool PAIRS, int POOL>
__global__ __launch_bounds__(kRopeThreads) void qk_norm_rope_kernel(RopeArgs a) {
  constexpr int LANES = D / 8;                 // of a token
  constexpr int GROUPS = kRopeThreads / LANES;  // tokens of a workgroup
  __shared__ float2 turns[GROUPS][D / 2];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int64_t tok = (int64_t)blockIdx.x * GROUPS + group;
  const bool live = tok < a.tokens;
  const int half = a.rot / 2;
  const int h0 = blockIdx.y * a.per_wg;
  const int h1 = h0 + a.per_wg < a.heads ? h0 + a.per_wg : a.heads;
  // a head's row, 16 bytes a lane: the next one is asked for before one is worked on, the
  // first before the turns are computed
  auto row_of = [&](int h) __attribute__((always_inline)) {
    const int which = h < a.hq ? 0 : (h < a.hq + a.hk ? 1 : 2);
    const int hh = h - (which == 0 ? 0 : (which == 1 ? a.hq : a.hq + a.hk));
    return ld16(a.src[which] + tok * a.token_stride[which] + hh * a.head_stride[which] + lane * 16);
  };
  u32x4 r = u32x4{0u, 0u, 0u, 0u};
  if (live) r = row_of(h0);
  if (live) {  // the token's turns: (cos, sin) of each frequency
    const double pos = (double)a.positions[tok];
    for (int i = lane; i < half; i += LANES) {
      const double f = a.freq64 ? reinterpret_cast<const double*>(a.inv_freq)[i]
                                : (double)reinterpret_cast<const float*>(a.inv_freq)[i];
      const double turn = pos * f * 0.15915494309189535;  // 1 / (2 pi)
      float s, c;
      sincospif((float)(2.0 * (turn - __builtin_rint(turn))), &s, &c);
      turns[group][i] = float2{c * a.rope_scale, s * a.rope_scale};
    }
  }
  __syncthreads();
  if (!live) return;
  // this lane's dims 8 * lane .. + 7: out = y * c + (partner's y) * s; the partner's dims are
  // half further on or back (halves), or its neighbours here (pairs); c = 1, s = 0 behind rot
  const int d0 = 8 * lane;
  const bool turned = d0 < a.rot;
  const bool back = !PAIRS && d0 >= half;      // (of a turned lane) the second half
  const int far = PAIRS ? 0 : (back ? -(half / 8) : half / 8);
  const int partner = turned ? lane + far : lane;
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int at = PAIRS ? d0 / 2 + i / 2 : d0 + i - (back ? half : 0);
    const float2 t = turned ? turns[group][at] : float2{1.f, 0.f};
    c[i] = t.x;
    s[i] = (PAIRS ? (i & 1) != 0 : back) ? t.y : -t.y;
  }
  int64_t slot = 0;
  bool store = true;
  if constexpr (POOL != kPoolNone) {
    slot = a.slots[tok];
    if (slot < 0 || slot >= a.num_slots) {  // -1 skips the token; anything else is an error
      if (slot != -1 && lane == 0 && blockIdx.y == 0) raise_err(a.err, MKV_DEVERR_SLOT);
      store = false;
    }
  }
  float w[8], wp[8];
  int have = -1;  // whose weights are held
  for (int h = h0; h < h1; ++h) {
    const int which = h < a.hq ? 0 : (h < a.hq + a.hk ? 1 : 2);
    const int hh = h - (which == 0 ? 0 : (which == 1 ? a.hq : a.hq + a.hk));
    u32x4 next = r;
    if (h + 1 < h1) next = row_of(h + 1);
    u32x4 out = r;
    if (which < 2) {
      const void* wt = a.weight[which];
      if (have != which && wt) {
        weights8(wt, a.weight_kind, a.centre, d0, w);
        weights8(wt, a.weight_kind, a.centre, 8 * partner, wp);
      }
      have = which;
      float x[8], xp[8];
      unpack8<F16>(r, x);
      float rstd = 1.f;
      if (wt) {
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += x[i] * x[i];
        rstd = 1.f / sqrtf(sum_lanes<LANES>(sq) / D + a.eps);
      }
      if constexpr (!PAIRS) {
        u32x4 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = (uint32_t)__shfl((int)r[i], partner, LANES);
        unpack8<F16>(p, xp);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= wt ? rstd * w[i] : 1.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (PAIRS) xp[i] = x[i ^ 1];
        else xp[i] *= wt ? rstd * wp[i] : 1.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        out[i] = pack2<F16>(turned ? x[2 * i] * c[2 * i] + xp[2 * i] * s[2 * i] : x[2 * i],
                            turned ? x[2 * i + 1] * c[2 * i + 1] + xp[2 * i + 1] * s[2 * i + 1]
                                   : x[2 * i + 1]);
    }
    r = next;
    if (which > 0 && !store) continue;
    // q and k leave past the caches (4096 tokens with the append 8.8 us instead of 9.7; 1021
    // of 15 heads of 128 5.6 instead of 6.0; an attention behind them takes as long either
    // way), the pool's 16-bit rows through them
    if (which == 0) {
      st_nt(a.q_out + (tok * a.hq + hh) * (2 * D) + lane * 16, out);
    } else if constexpr (POOL == kPoolNone) {
      st_nt(a.k_out + (tok * a.hk + hh) * (2 * D) + lane * 16, out);
    } else {
      const int64_t row = slot * a.hk + hh;
      uint8_t* pool = a.pool[which - 1];
      if constexpr (POOL == kPool16) {
        st16(pool + row * (2 * D) + lane * 16, out);
      } else {
        const uint32_t o[4] = {out[0], out[1], out[2], out[3]};
        if constexpr (POOL == kPoolFp8) {
          uint32_t codes[2];
          const float scale = quantise_fp8<LANES, 8>(o, codes);
          *reinterpret_cast<u32x2*>(pool + row * D + lane * 8) = u32x2{codes[0], codes[1]};
          if (lane == 0) a.scale[which - 1][row] = scale;
        } else {
          uint32_t codes[1];
          const uint32_t byte = quantise_fp4<8>(o, codes);
          *reinterpret_cast<uint32_t*>(pool + row * kFp4Row + lane * 4) = codes[0];
          if ((lane & 3) == 0) pool[row * kFp4Row + kFp4Codes + lane / 4] = (uint8_t)byte;
        }
      }
    }
  }
}

// Workgroups for the tokens: dim / 8 lanes own a token.
int64_t workgroups(int64_t tokens, int32_t dim) {
  const int64_t groups = kRopeThreads / (dim / 8);
  return (tokens + groups - 1) / groups;
}

template <int D, bool F16, bool PAIRS, int POOL>
void launch(RopeArgs& a, hipStream_t st) {
  const int64_t wgs = workgroups(a.tokens, D);
  // a token's heads over several workgroups while the tokens alone are few: up to 4 for each
  // CU (4096 tokens of 6 heads with the append: 8.8 us, with up to 2 10.4, with up to 8 8.7)
  const int64_t want = 4ll * device_cus();
  int64_t split = (want + wgs - 1) / wgs;
  split = split > a.heads ? a.heads : split;
  a.per_wg = (int32_t)((a.heads + split - 1) / split);
  hipLaunchKernelGGL((qk_norm_rope_kernel<D, F16, PAIRS, POOL>),
                     dim3((unsigned)wgs, (unsigned)((a.heads + a.per_wg - 1) / a.per_wg)),
                     dim3(kRopeThreads), 0, st, a);
}

template <bool F16, bool PAIRS, int POOL>
void launch_dim(int32_t dim, RopeArgs& a, hipStream_t st) {
  if constexpr (POOL == kPoolFp8 || POOL == kPoolFp4) {
    launch<256, F16, PAIRS, POOL>(a, st);
  } else {
    if (dim == 64) launch<64, F16, PAIRS, POOL>(a, st);
    else if (dim == 128) launch<128, F16, PAIRS, POOL>(a, st);
    else launch<256, F16, PAIRS, POOL>(a, st);
  }
}

template <bool F16, int POOL>
void launch_style(int32_t dim, bool pairs, RopeArgs& a, hipStream_t st) {
  if (pairs) launch_dim<F16, true, POOL>(dim, a, st);
  else launch_dim<F16, false, POOL>(dim, a, st);
}

template <int POOL>
void launch_type(int32_t dim, bool f16, bool pairs, RopeArgs& a, hipStream_t st) {
  if constexpr (POOL == kPoolFp8 || POOL == kPoolFp4) {
    launch_style<false, POOL>(dim, pairs, a, st);
  } else {
    if (f16) launch_style<true, POOL>(dim, pairs, a, st);
    else launch_style<false, POOL>(dim, pairs, a, st);
  }
}

// Argument checks and fields shared by the two entry points.
int fill(const char* fn, RopeArgs& a, const void* q, int64_t q_token, int64_t q_head, const void* k,
         int64_t k_token, int64_t k_head, int64_t tokens, int32_t hq, int32_t hk, int32_t dim,
         const int64_t* positions, const void* inv_freq, int32_t freq64, int32_t rot,
         float rope_scale, const void* q_weight, const void* k_weight, int32_t weight_kind,
         int32_t zero_centered, float eps, void* q_out) {
  MKV_REQUIRE(tokens >= 0 && hq >= 0 && hk >= 0, MKV_E_INVALID, "%s: bad size", fn);
  MKV_REQUIRE(dim == 64 || dim == 128 || dim == 256, MKV_E_UNSUPPORTED,
              "%s: head_dim %d unsupported (64, 128, 256)", fn, dim);
  MKV_REQUIRE(rot > 0 && rot <= dim && rot % 16 == 0, MKV_E_UNSUPPORTED,
              "%s: rotary dim %d unsupported (multiples of 16 up to head_dim)", fn, rot);
  MKV_REQUIRE(hq <= 65536 && hk <= 65536 && tokens < (1ll << 31) &&
                  grid_fits(workgroups(tokens, dim), kRopeThreads),
              MKV_E_UNSUPPORTED, "%s: too many rows for one call", fn);
  MKV_REQUIRE(weight_kind >= kNoWeight && weight_kind <= kWeightF32, MKV_E_INVALID,
              "%s: bad weight type", fn);
  if (tokens == 0 || hq + hk == 0) return MKV_OK;
  MKV_REQUIRE((hq == 0 || (q && q_out)) && (hk == 0 || k) && positions && inv_freq, MKV_E_INVALID,
              "%s: null pointer", fn);
  MKV_REQUIRE(aligned16(q) && aligned16(k) && aligned16(q_out) && aligned16(q_weight) &&
                  aligned16(k_weight) && q_token % 16 == 0 && q_head % 16 == 0 &&
                  k_token % 16 == 0 && k_head % 16 == 0,
              MKV_E_ALIGN, "%s: misaligned pointer or stride", fn);
  MKV_REQUIRE(((uintptr_t)inv_freq & (freq64 ? 7 : 3)) == 0 && ((uintptr_t)positions & 7) == 0,
              MKV_E_ALIGN, "%s: misaligned positions or inv_freq", fn);
  a = RopeArgs{};
  a.src[0] = (const uint8_t*)q;
  a.src[1] = (const uint8_t*)k;
  a.token_stride[0] = q_token;
  a.token_stride[1] = k_token;
  a.head_stride[0] = q_head;
  a.head_stride[1] = k_head;
  a.q_out = (uint8_t*)q_out;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.weight[0] = weight_kind == kNoWeight ? nullptr : q_weight;
  a.weight[1] = weight_kind == kNoWeight ? nullptr : k_weight;
  a.tokens = tokens;
  a.hq = hq;
  a.hk = hk;
  a.rot = rot;
  a.freq64 = freq64;
  a.weight_kind = weight_kind;
  a.eps = eps;
  a.rope_scale = rope_scale;
  a.centre = zero_centered ? 1.f : 0.f;
  return MKV_OK;
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" int mkv_qk_norm_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                const void* k, int64_t k_token_stride, int64_t k_head_stride,
                                int64_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads,
                                int32_t head_dim, int32_t fp16, const int64_t* positions,
                                const void* inv_freq, int32_t freq_fp64, int32_t rotary_dim,
                                int32_t interleaved, float rope_scale, const void* q_weight,
                                const void* k_weight, int32_t weight_type, int32_t zero_centered,
                                float eps, void* q_out, void* k_out, void* stream) {
  static const char* fn = "mkv_qk_norm_rope";
  clear_error();
  RopeArgs a;
  const int rc = fill(fn, a, q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride,
                      num_tokens, num_q_heads, num_kv_heads, head_dim, positions, inv_freq,
                      freq_fp64, rotary_dim, rope_scale, q_weight, k_weight, weight_type,
                      zero_centered, eps, q_out);
  if (rc != MKV_OK) return rc;
  if (num_tokens == 0 || num_q_heads + num_kv_heads == 0) return MKV_OK;
  MKV_REQUIRE(num_kv_heads == 0 || k_out, MKV_E_INVALID, "%s: null pointer", fn);
  MKV_REQUIRE(aligned16(k_out), MKV_E_ALIGN, "%s: misaligned pointer or stride", fn);
  a.k_out = (uint8_t*)k_out;
  a.heads = num_q_heads + num_kv_heads;
  launch_type<kPoolNone>(head_dim, fp16 != 0, interleaved != 0, a, as_stream(stream));
  return check_launch(fn);
}

extern "C" int mkv_append_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                               const void* k, int64_t k_token_stride, int64_t k_head_stride,
                               const void* v, int64_t v_token_stride, int64_t v_head_stride,
                               int64_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads,
                               int32_t head_dim, int32_t fp16, const int64_t* positions,
                               const void* inv_freq, int32_t freq_fp64, int32_t rotary_dim,
                               int32_t interleaved, float rope_scale, const void* q_weight,
                               const void* k_weight, int32_t weight_type, int32_t zero_centered,
                               float eps, void* q_out, int32_t pool_type, void* k_pool,
                               void* v_pool, float* k_scale, float* v_scale, int64_t num_slots,
                               const int64_t* slot_mapping, int32_t* err, void* stream) {
  static const char* fn = "mkv_append_rope";
  clear_error();
  RopeArgs a;
  const int rc = fill(fn, a, q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride,
                      num_tokens, num_q_heads, num_kv_heads, head_dim, positions, inv_freq,
                      freq_fp64, rotary_dim, rope_scale, q_weight, k_weight, weight_type,
                      zero_centered, eps, q_out);
  if (rc != MKV_OK) return rc;
  MKV_REQUIRE(num_kv_heads > 0 && num_slots >= 0, MKV_E_INVALID, "%s: bad size", fn);
  MKV_REQUIRE(pool_type >= kPool16 && pool_type <= kPoolFp4, MKV_E_INVALID, "%s: bad pool type", fn);
  MKV_REQUIRE(pool_type == kPool16 || (head_dim == 256 && !fp16), MKV_E_UNSUPPORTED,
              "%s: fp8 and 4-bit pools take bf16 heads of 256", fn);
  if (num_tokens == 0) return MKV_OK;
  MKV_REQUIRE(v && k_pool && v_pool && slot_mapping && err &&
                  (pool_type != kPoolFp8 || (k_scale && v_scale)),
              MKV_E_INVALID, "%s: null pointer", fn);
  MKV_REQUIRE(aligned16(v) && v_token_stride % 16 == 0 && v_head_stride % 16 == 0 &&
                  aligned16(k_pool) && aligned16(v_pool) && aligned4(k_scale) &&
                  aligned4(v_scale) && ((uintptr_t)slot_mapping & 7) == 0,
              MKV_E_ALIGN, "%s: misaligned pointer or stride", fn);
  a.src[2] = (const uint8_t*)v;
  a.token_stride[2] = v_token_stride;
  a.head_stride[2] = v_head_stride;
  a.pool[0] = (uint8_t*)k_pool;
  a.pool[1] = (uint8_t*)v_pool;
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.num_slots = num_slots;
  a.slots = slot_mapping;
  a.err = err;
  a.heads = num_q_heads + 2 * num_kv_heads;
  const hipStream_t st = as_stream(stream);
  if (pool_type == kPool16)
    launch_type<kPool16>(head_dim, fp16 != 0, interleaved != 0, a, st);
  else if (pool_type == kPoolFp8)
    launch_type<kPoolFp8>(head_dim, false, interleaved != 0, a, st);
  else
    launch_type<kPoolFp4>(head_dim, false, interleaved != 0, a, st);
  return check_launch(fn);
}
