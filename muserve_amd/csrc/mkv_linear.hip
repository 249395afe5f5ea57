// mkv_linear.hip — linear attention with a decay for each head over the state
// pool (gfx950): the recurrent form for single tokens, the form for packed
// prompts, and the gated RMS norm behind both.
//
// A value head's state is S [128 values, 128 keys] fp32, one per request slot.
// A token with key k, query q, value v, log decay g and, for the delta rule, a
// write strength beta does
//     S <- e^g S,   u = beta (v - S k)   (u = v without beta),
//     S <- S + u k^T,   o = scale S q,
// with q and k divided by sqrt(|.|^2 + 1e-6) first where asked. Value head h
// reads key head h / (num_v_heads / num_k_heads). The rows of S (one per value
// dim) never meet, so they are spread over threads, waves and workgroups.
#include <math.h>

#include "mkv_device.h"

namespace mkv {
namespace {

constexpr int kDim = 128;             // key and value dims of a head
constexpr float kL2Eps = 1e-6f;       // of the q and k norms
constexpr int64_t kStateHead = (int64_t)kDim * kDim;  // floats of a head's state

struct LinArgs {
  float* state;  // [pool_slots, hv, 128, 128], values x keys
  int64_t pool_slots;
  const int32_t* slots;  // [n], unique
  int32_t n;             // requests (decode) or sequences
  int32_t hk, hv, group; // heads, and value heads per key head
  const uint8_t *q, *k, *v;  // bf16 rows, strides in bytes between tokens
  int64_t q_stride, k_stride, v_stride;
  const uint8_t *g, *beta;  // [tokens, hv], fp32 or bf16; beta null: no delta rule
  int64_t g_stride, beta_stride;
  int32_t gates_bf16;
  const float *a_log, *dt_bias;  // [hv]: g and beta are projections (both null: final values)
  int32_t qk_norm;
  float scale;
  const uint8_t *z, *w;  // the output norm's gate [tokens, hv, 128] bf16 and weight; null: none
  int64_t z_stride;
  int32_t w_bf16;
  float eps;
  uint8_t* out;       // [tokens, hv, 128] bf16
  const int32_t* cu;  // prompts: [n + 1]
  int64_t tokens;
  int32_t* err;
};

__device__ __forceinline__ float bf16_at(const uint8_t* p) {
  return bits_f32((uint32_t) * (const uint16_t*)p << 16);
}
__device__ __forceinline__ float gate_at(const uint8_t* p, int32_t bf16, int64_t i) {
  return bf16 ? bf16_at(p + 2 * i) : *(const float*)(p + 4 * i);
}
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// A token's log decay and write strength for value head h. Projections a and b
// become -e^a_log softplus(a + dt_bias) and sigmoid(b).
__device__ __forceinline__ void load_gates(const LinArgs& a, int64_t token, int32_t h, float& g,
                                           float& beta) {
  g = gate_at(a.g + token * a.g_stride, a.gates_bf16, h);
  beta = a.beta ? gate_at(a.beta + token * a.beta_stride, a.gates_bf16, h) : 1.f;
  if (a.a_log) {
    const float x = g + a.dt_bias[h];
    g = -expf(a.a_log[h]) * ((x < 0.f ? 0.f : x) + log1pf(expf(-fabsf(x))));  // (NaN stays)
    if (a.beta) beta = sigmoid(beta);
  }
}

// 4 consecutive bf16
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void unpack4(u32x2 w, float (&x)[4]) {
  x[0] = bits_f32(w.x << 16);
  x[1] = bits_f32(w.x & 0xffff0000u);
  x[2] = bits_f32(w.y << 16);
  x[3] = bits_f32(w.y & 0xffff0000u);
}
__device__ __forceinline__ void load4(const uint8_t* p, float (&x)[4]) {
  unpack4(*(const u32x2*)p, x);
}

// The recurrence over a few tokens with a head's state in registers: a row of
// S is 8 lanes x 16 floats (lane l holds columns 4 l + 32 c .. +3, whole
// 128-byte lines per 8 lanes), a thread holds ROWS rows. S k and S q are both
// taken of the old state, so that their sums over lanes run together:
//     o = scale (e^g S q + u (k . q)).
template <int ROWS>
struct Rows {
  float s[ROWS][16];
  float kx[16], qx[16];
  float rk, rq, kq;  // 1 / norms, and k . q with them

  // this lane's columns of a token's k and q, and the sums over them
  __device__ __forceinline__ void keys(const LinArgs& a, int64_t token, int32_t kh, int l) {
    const uint8_t* kp = a.k + token * a.k_stride + kh * (kDim * 2) + l * 8;
    const uint8_t* qp = a.q + token * a.q_stride + kh * (kDim * 2) + l * 8;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float x[4], y[4];
      load4(kp + 64 * c, x);
      load4(qp + 64 * c, y);
#pragma unroll
      for (int j = 0; j < 4; ++j) kx[4 * c + j] = x[j], qx[4 * c + j] = y[j];
    }
  }
  __device__ __forceinline__ void norms(const LinArgs& a) {
    float kk = 0.f, qq = 0.f, m = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      kk = fmaf(kx[j], kx[j], kk);
      qq = fmaf(qx[j], qx[j], qq);
      m = fmaf(kx[j], qx[j], m);
    }
    m = sum_lanes<8>(m);
    rk = rq = 1.f;
    if (a.qk_norm) {
      rk = 1.f / sqrtf(sum_lanes<8>(kk) + kL2Eps);
      rq = 1.f / sqrtf(sum_lanes<8>(qq) + kL2Eps);
    }
    kq = m * rk * rq;
  }
  // one token; v: this thread's values, o: its outputs (all 8 lanes of a row)
  __device__ __forceinline__ void step(const LinArgs& a, float g, float beta, const float (&v)[ROWS],
                                       float (&o)[ROWS]) {
    const float e = expf(g);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        x = fmaf(s[i][j], kx[j], x);
        y = fmaf(s[i][j], qx[j], y);
      }
      x = sum_lanes<8>(x);
      y = sum_lanes<8>(y);
      const float u = a.beta ? beta * (v[i] - e * rk * x) : v[i];
      o[i] = a.scale * (e * rq * y + u * kq);
      const float w = u * rk;
#pragma unroll
      for (int j = 0; j < 16; ++j) s[i][j] = fmaf(w, kx[j], e * s[i][j]);
    }
  }
};

__device__ __forceinline__ float weight_at(const uint8_t* w, int32_t bf16, int64_t i) {
  return bf16 ? bf16_at(w + 2 * i) : *(const float*)(w + 4 * i);
}

// o / sqrt(mean(o^2) + eps) w silu(z) of a head whose 128 dims a workgroup of 4 waves
// has, dims r0 + 32 i in the 8 lanes l of a row; part: a float for each wave.
template <int ROWS>
__device__ __forceinline__ void norm_over_dims(const LinArgs& a, int64_t token, int32_t h, int r0,
                                               int l, float* part, float (&o)[ROWS]) {
  static_assert(ROWS * 32 == kDim && kThreads == 256, "a head");
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) q = fmaf(o[i], o[i], q);
  q = sum_lanes<64>(l == 0 ? q : 0.f);  // (8 lanes have the same rows)
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = q;
  __syncthreads();
  q = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) q += part[i];
  const float r = 1.f / sqrtf(q * (1.f / kDim) + a.eps);
  const uint8_t* zp = a.z + token * a.z_stride + h * (kDim * 2);
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int d = r0 + 32 * i;
    o[i] = o[i] * r * weight_at(a.w, a.w_bf16, d) * silu_bf16(bf16_at(zp + 2 * d));
  }
}

// One workgroup per (value head, request): the head's 64 KiB state is read
// once, updated in registers and written back. Bound by HBM: 128 KiB per
// (request, head) against 0.8 KiB of everything else; 256 requests of 8 heads
// take 53 us, 5.1 TB/s. A lone request (7.0 us) is bound by its two trips to
// memory: 1024 threads a head, with 4 rows' loads less each, were no faster.
__global__ __launch_bounds__(kThreads) void linear_decode_kernel(LinArgs a) {
  constexpr int kGroups = kThreads / 8, kRows = kDim / kGroups;
  const int tid = threadIdx.x, l = tid & 7, r0 = tid >> 3;
  const int32_t h = blockIdx.x, kh = h / a.group;
  const int64_t b = blockIdx.y;
  const int32_t slot = ld_const(a.slots + b);
  uint8_t* out = a.out + (b * a.hv + h) * (kDim * 2);
  if (slot < 0 || slot >= a.pool_slots) {  // uniform
    if (h == 0 && tid == 0) raise_err(a.err, MKV_DEVERR_STATE_SLOT);
    if (tid < kDim / 2) *(uint32_t*)(out + 4 * tid) = 0u;
    return;
  }
  float* st = a.state + ((int64_t)slot * a.hv + h) * kStateHead;
  Rows<kRows> m;
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const u32x4 x = ld_nt((const uint8_t*)(st + (r0 + kGroups * i) * kDim + 32 * c + 4 * l));
#pragma unroll
      for (int j = 0; j < 4; ++j) m.s[i][4 * c + j] = bits_f32(x[j]);
    }
  m.keys(a, b, kh, l);
  float g, beta, v[kRows], o[kRows];
  load_gates(a, b, h, g, beta);
  const uint8_t* vp = a.v + b * a.v_stride + h * (kDim * 2);
#pragma unroll
  for (int i = 0; i < kRows; ++i) v[i] = bf16_at(vp + 2 * (r0 + kGroups * i));
  m.norms(a);
  m.step(a, g, beta, v, o);
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u32x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = f32_bits(m.s[i][4 * c + j]);
      st_stream((uint8_t*)st, (uint32_t)((r0 + kGroups * i) * kDim + 32 * c + 4 * l) * 4, x);
    }
  __shared__ float part[kThreads / 64];
  if (a.z) norm_over_dims<kRows>(a, b, h, r0, l, part, o);  // uniform
  if (l == 0) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      *(uint16_t*)(out + 2 * (r0 + kGroups * i)) = f32_to_bf16_rne(o[i]);
  }
}

// ---------------------------------------------------------------------------
// Prompts
// ---------------------------------------------------------------------------

// One workgroup per 64 value dims of a (head, sequence), or per 128 with the output
// norm, which needs them all, token after token: bound by the chain from one to the
// next, 1.8 us each while few workgroups run.
template <bool NORM>
__global__ __launch_bounds__(256) void linear_scan_kernel(LinArgs a) {
  constexpr int kRows = NORM ? 4 : 2, kParts = 4 / kRows;
  const int tid = threadIdx.x, l = tid & 7, r0 = tid >> 3;
  const int32_t h = blockIdx.x / kParts, kh = h / a.group, d0 = blockIdx.x % kParts * 64;
  const int32_t b = blockIdx.y;
  const bool first = blockIdx.x == 0 && tid == 0;
  if (!offsets_ok(a.cu, a.n, a.tokens)) {
    if (first && b == 0) raise_err(a.err, MKV_DEVERR_TABLE);
    return;
  }
  const int64_t t0 = a.cu[b], t1 = a.cu[b + 1];
  if (t0 == t1) return;  // uniform
  const int32_t slot = a.slots[b];
  if (slot < 0 || slot >= a.pool_slots) {  // uniform
    if (first) raise_err(a.err, MKV_DEVERR_STATE_SLOT);
    constexpr int kWords = kRows * 16;  // of a token's dims
    for (int64_t t = t0 + tid / kWords; t < t1; t += 256 / kWords)
      *(uint32_t*)(a.out + (t * a.hv + h) * (kDim * 2) + d0 * 2 + 4 * (tid % kWords)) = 0u;
    return;
  }
  float* st = a.state + ((int64_t)slot * a.hv + h) * kStateHead + (int64_t)d0 * kDim;
  Rows<kRows> m;
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const u32x4 x = ld16((const uint8_t*)(st + (r0 + 32 * i) * kDim + 32 * c + 4 * l));
#pragma unroll
      for (int j = 0; j < 4; ++j) m.s[i][4 * c + j] = bits_f32(x[j]);
    }
  __shared__ float part[2][4];
  for (int64_t t = t0; t < t1; ++t) {
    float g, beta, v[kRows], o[kRows];
    m.keys(a, t, kh, l);
    load_gates(a, t, h, g, beta);
    const uint8_t* vp = a.v + t * a.v_stride + (h * kDim + d0) * 2;
#pragma unroll
    for (int i = 0; i < kRows; ++i) v[i] = bf16_at(vp + 2 * (r0 + 32 * i));
    m.norms(a);
    m.step(a, g, beta, v, o);
    if constexpr (NORM)  // (the last token's sums may still be read)
      norm_over_dims<kRows>(a, t, h, r0, l, part[(t - t0) & 1], o);
    if (l == 0) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        *(uint16_t*)(a.out + ((t * a.hv + h) * kDim + d0 + r0 + 32 * i) * 2) =
            f32_to_bf16_rne(o[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u32x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = f32_bits(m.s[i][4 * c + j]);
      st16((uint8_t*)(st + (r0 + 32 * i) * kDim + 32 * c + 4 * l), x);
    }
}

// ---------------------------------------------------------------------------
// Prompts in chunks of 64 tokens, on the matrix cores. With G_i the sum of a
// chunk's log decays up to token i, k and q normalised, S0 the state before it:
//     A_ij = beta_i e^(G_i - G_j) k_i . k_j   (j < i),   T = (I + A)^-1
//     U = T diag(beta) (V - diag(e^G) K S0^T) (U = V without the delta rule)
//     O = scale (diag(e^G) Q S0^T + P U),     P_ij = e^(G_i - G_j) q_i . k_j  (j <= i)
//     S = e^G_63 S0 + sum_j e^(G_63 - G_j) u_j k_j^T
// linear_prep_kernel makes what does not depend on the state (T, P and the
// factors of each token), for all chunks at once; linear_chunk_kernel walks a
// sequence's chunks with the state in registers.
//
// Precision: the matrix instructions of a chunk take fp16. Rows of k and q are
// brought near 1 by a power of two, which the factors of their tokens undo: a
// bf16 row is exact in fp16 then, but for elements below 2^-17 of its largest,
// rounded to 2^-25 of that. An fp32 operand (the state, the right-hand side, T, u, P)
// is two fp16 parts, 22 bits; the product of two such drops the lower parts' (2^-22).
// Sums run in fp32 in the matrix cores. So a state and an output before its rounding
// to bf16 are within a few 2^-22 of what they are sums of (600 tokens: states 1.4e-7
// from float64 in the norm, 1.0e-7 token by token; outputs 1.66e-3 both). (With one part of the
// state, P and u in the outputs these were 2^-12 of their terms off, which shows where
// terms cancel; 28 matrix instructions of 132 a chunk, 3 to 6 % of a call.) Three bf16
// parts were as exact as fp32, but take 182 matrix and 630 vector instructions a chunk.
//
// Scale: two fp16 parts end at 2^-25, so what is small beside what else an operand
// holds is lost there. A value dim's state (a column of the operands, which never mixes
// with another) is kept times a power of two f of its own, and its values go in times f
// too. Before a chunk f goes by the dim's state, or by its values where these make the
// dim's new state, as the chunk's decays leave little of the old: the step is then 2^-28
// of them or less. What is left are the tokens of a dim in one chunk. Where some stand
// far above the rest, and decays leave nothing of them, the rest is exact to 2^-28 of
// the larger only; where that is too little (values of 4 tokens in a row below 2^-13 of
// it), the chunk is walked token by token. (One f for a wave's 16 dims left a dim of
// 2^-20 of the largest without a digit, and f by the state alone the values behind a
// forgotten state of 2^20 of them. f by dim and chunk costs 2 to 6 % of a call.)
//
// The rows (tokens) of a chunk mix also through zeros. So that what is out of the
// ordinary in one token (infinities, NaN) reaches only the tokens after it, such a
// chunk is walked token by token as well: inputs past 2^60 in size, a chunk whose
// decays grow by more than e^2 (where products could overflow and the recurrence not),
// operands past the limits below.
// ---------------------------------------------------------------------------
typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4;
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
typedef __attribute__((address_space(3))) float lds_f32;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kChunk = 64;
// Operand images: blocks of 1 KiB, 16 bytes per lane, one v_mfma_f32_16x16x32
// A operand each. Lane (m = lane % 16, d = lane / 16) has row m, columns
// 32 s + 16 (j / 4) + 4 d + j % 4, j = 0 .. 7: the order in which a lane holds
// the rows of two 16 x 16 results, so that results are B operands as they lie.
constexpr int kFrag = 1024;
constexpr int kKeyImage = 48 * kFrag;  // of a chunk's key head: K, Q (4 row blocks x 4), K^T (8 x 2)
constexpr int kLower = 6;              // operands of a 64 x 64 lower triangle
constexpr int kTParts = 2, kPParts = 2;
// The factors of a chunk's tokens, [64] each: of K S0^T in the right-hand side,
// of u in the state, e^G, of the output, of v; then e^G_63, the largest factor of v,
// whether to walk (two words), and log2 of e^G.
constexpr int kFactors = 2048, kFacX = 0, kFacU = 64, kFacG = 128, kFacO = 192, kFacV = 256;
constexpr int kFacAll = 320, kFacMax = 321, kFacWalk = 322, kFacLog = 384;
constexpr int head_image(bool delta) {
  return (delta ? kTParts * kLower * kFrag : 0) + kPParts * kLower * kFrag + kFactors;
}
__device__ __forceinline__ constexpr int lower(int mt, int s) {  // operand of rows 16 mt, step s
  return mt < 2 ? mt : mt < 3 ? 2 + s : 4 + s;
}
constexpr uint32_t kHugeBf16 = (127 + 60) << 7;  // k, q: |x| >= 2^60, infinities and NaN
constexpr double kLeastDecay = -1e5;             // e^g is 0 far above it; -inf would make NaN sums
constexpr float kMostPart = 0x1p15f;  // of operands of fp16 parts (fp16 ends at 2^16)
constexpr float kMostRhs = 0x1p10f;   // of right-hand sides, in units of the dim's scale
constexpr float kMostState = 0x1p14f;
// T and P are held times these, which the factors of u in the state and of the
// output undo (and e^G has): the fp16 step under a small element is less of a large
// one.
constexpr float kTScale = 0x1p4f, kPScale = 0x1p6f;
// A dim's scale before a chunk holds the largest of its state, or of its values where
// the chunk leaves the state below kLittle of them (or they are past kHighValue), in
// these bounds, else it is brought to 2^kNearState or 2^kNearValue.
constexpr float kLittle = 0x1p-5f;
constexpr float kLowState = 0x1p3f, kHighState = 0x1p6f, kLowValue = 0x1p4f, kHighValue = 0x1p8f;
constexpr int kNearState = 4, kNearValue = 6;
// Too coarse is what the values of 4 tokens in a row do to a dim in such a chunk, if it
// is less than kLeastQuad of its largest right-hand side and nothing larger of what was
// before is left by then, or there are kManyQuads of them (the few others stand out);
// and all it does, where the state is left below kLeastState of itself, and the values
// are below kLeastValue of it.
constexpr float kLeastQuad = 0x1p-13f, kLeastState = 0x1p-10f, kLeastValue = 0x1p-9f;
constexpr int kManyQuads = 4;

constexpr int64_t kMostStride = 1 << 24;  // 64 rows through a buffer descriptor

constexpr uint32_t kXcds = 8;

struct ChunkArgs {
  uint8_t* keys;   // [ids][khs] key images
  uint8_t* heads;  // [ids][khs * group] head images
  int32_t kh0, khs;  // key heads of this launch
  int32_t parts;     // workgroups per head
  int32_t rows;      // sequences, or segments
  int32_t seg;       // tokens of a segment (a multiple of 64)
  float* ends;       // [segment ids][heads of the launch][128][128]: B, then the first states
  float* steps;      // as ends: M's operand blocks; without the delta rule one factor each
};

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p;
}
__device__ __forceinline__ u32x4 lds_ld16(uint32_t at) { return *(lds_u32x4*)(uintptr_t)at; }
__device__ __forceinline__ void lds_st16(uint32_t at, u32x4 v) { *(lds_u32x4*)(uintptr_t)at = v; }
__device__ __forceinline__ f32x4 lds_ldf4(uint32_t at) {
  return __builtin_bit_cast(f32x4, lds_ld16(at));
}
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ f32x4 mfma(u32x4 x, u32x4 y, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x),
                                                 __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma16(u32x4 x, u32x4 y, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x),
                                                __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t f16_pack(float lo, float hi) {  // to nearest even
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, f16x2));
}
// 8 floats in fp16; cut: and what that leaves of them (exact)
__device__ __forceinline__ u32x4 upper(const float (&x)[8]) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = f16_pack(x[2 * i], x[2 * i + 1]);
  return w;
}
__device__ __forceinline__ u32x4 cut(float (&x)[8]) {
  const u32x4 w = upper(x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // x - half: one mixed fma each (the compiler converts and subtracts)
    const uint32_t h = w[i];
    float lo, hi;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(lo) : "v"(h), "v"(x[2 * i]));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(hi)
        : "v"(h), "v"(x[2 * i + 1]));
    x[2 * i] = lo;
    x[2 * i + 1] = hi;
  }
  return w;
}
// max(m, |x|, |y|): a NaN among them is passed over, or (any_of) is the result. One
// instruction each, in the compiler's hands: it waits for matrix results that they
// read, and before a lane reads what another has of theirs. (As inline assembly they
// had read matrix results one instruction behind.) The empty assembly keeps them in
// their places, or values would wait for them in registers that there are not.
__device__ __forceinline__ float any_of(float m, float x, float y) {
  m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(m, fabsf(x)), fabsf(y));
  asm("" : "+v"(m));
  return m;
}
__device__ __forceinline__ float most_of(float m, float x, float y) {
  m = fmaxf(fmaxf(m, fabsf(x)), fabsf(y));
  asm("" : "+v"(m));
  return m;
}

// e^x of a difference of running sums. They are float64: sums far from 0 have
// small differences. The result's error is |x| e^x 2^-24, at most 0.4 steps of 1.
__device__ __forceinline__ float exp_of(double x) {
  return __builtin_amdgcn_exp2f((float)(x * 1.4426950408889634074));
}

// x of the lane that a row shift or broadcast (as a DPP control) names, 0 where
// there is none or a row of 16 lanes is not among ROWS
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double lanes_below(double x) {
  const u32x2 w = __builtin_bit_cast(u32x2, x);
  const uint32_t lo = w.x, hi = w.y;
  return __builtin_bit_cast(
      double, u32x2{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)lo, CTRL, ROWS, 0xf, true),
                    (uint32_t)__builtin_amdgcn_update_dpp(0, (int)hi, CTRL, ROWS, 0xf, true)});
}
__device__ __forceinline__ double lane_at(double x, int lane) {
  const u32x2 w = __builtin_bit_cast(u32x2, x);
  const uint32_t lo = w.x, hi = w.y;
  return __builtin_bit_cast(double,
                            u32x2{(uint32_t)__builtin_amdgcn_readlane((int)lo, lane),
                                  (uint32_t)__builtin_amdgcn_readlane((int)hi, lane)});
}

__device__ __forceinline__ bool huge(u32x4 w) {  // any of 8 bf16
  bool h = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h |= (w[i] & 0x7f80u) >= kHugeBf16 || ((w[i] >> 16) & 0x7f80u) >= kHugeBf16;
  return h;
}

// One workgroup per (chunk, key head): K and Q rows through LDS, their images;
// then the value heads of the group, four at a time: a wave makes a head's P and
// factors, and with the delta rule another one A and T. That wave keeps A as 10
// 16 x 16 blocks in LDS (row-major, 16-byte chunks XORed by row / 4) and inverts
// by blocks: the diagonal ones by forward substitution, a lane per column, the
// rest in fp32 matrix instructions (16x16x4). Bound by the latency of these
// chains: 512 chunks of 8 heads take 45 us, a lone one 13 (of which 6 until the
// rows are staged, 6.5 A and T); with one wave for both parts of a head (2 waves
// per SIMD, not 4) 48 and 17. K's rows all in registers would spill (70 us).
constexpr int kRowB = 272;  // bytes of a staged row: 256 and a pad against bank conflicts
constexpr int kBlocks = 10;
constexpr int kSlots = 4;   // heads at a time

template <bool DELTA>
__global__ __launch_bounds__(DELTA ? 512 : 256, 4) void linear_prep_kernel(LinArgs a, ChunkArgs c) {
  constexpr int kWaves = DELTA ? 8 : 4;
  __shared__ __attribute__((aligned(16))) uint8_t stage[2 * kChunk * kRowB];
  __shared__ __attribute__((aligned(16))) uint8_t blocks[kSlots][DELTA ? kBlocks * kFrag : 16];
  __shared__ double run[kSlots][kChunk];
  // e^(G_16 mt - G_j) for j < 16 mt: 16, 32 and 48 of them
  __shared__ __attribute__((aligned(16))) float since[kSlots][96];
  __shared__ float inv[2][kChunk];   // 1 / norms of k, q
  // the powers of two that bring rows of k, q near 1
  __shared__ __attribute__((aligned(16))) float unit[2][kChunk];
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, d = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t id = blockIdx.x;
  const int32_t kh = c.kh0 + blockIdx.y;
  int64_t s0 = 0, s1 = 0, t0 = 0;
  if (tile_sequence(a.cu, a.n, a.tokens, id, kChunk, s0, s1, t0) < 0) return;  // uniform
  const int32_t len = (int32_t)(s1 - t0 < kChunk ? s1 - t0 : kChunk);

  // lane i has token i's gates; their loads run with the first rows'
  const int slot = wave & (kSlots - 1);
  const bool makes_t = wave >= kSlots;  // uniform
  float g = 0.f, beta = 0.f;
  u32x4 rows[2][16 / kWaves];
#pragma unroll
  for (int u = 0; u < 16 / kWaves; ++u) {  // 16 chunks of 16 bytes per row
    const int r = (tid >> 4) + 4 * kWaves * u, ch = tid & 15;
    rows[0][u] = rows[1][u] = u32x4{0u, 0u, 0u, 0u};
    if (r < len) {
      rows[0][u] = ld16(a.k + (t0 + r) * a.k_stride + kh * (kDim * 2) + ch * 16);
      rows[1][u] = ld16(a.q + (t0 + r) * a.q_stride + kh * (kDim * 2) + ch * 16);
    }
  }
  if (slot < a.group && lane < len) load_gates(a, t0 + lane, kh * a.group + slot, g, beta);
  bool odd = false;
#pragma unroll
  for (int u = 0; u < 16 / kWaves; ++u) {
    const int r = (tid >> 4) + 4 * kWaves * u, ch = tid & 15;
    const u32x4 kv = rows[0][u], qv = rows[1][u];
    odd |= huge(kv) || huge(qv);
    *(u32x4*)(stage + r * kRowB + ch * 16) = kv;
    *(u32x4*)(stage + (kChunk + r) * kRowB + ch * 16) = qv;
    float kk = 0.f, qq = 0.f;
    uint32_t ke = 37u << 7, qe = ke;  // largest exponents (as bf16), from 2^-90 up
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ke = max(ke, max(kv[i] & 0x7f80u, (kv[i] >> 16) & 0x7f80u));
      qe = max(qe, max(qv[i] & 0x7f80u, (qv[i] >> 16) & 0x7f80u));
      const float k0 = bits_f32(kv[i] << 16), k1 = bits_f32(kv[i] & 0xffff0000u);
      const float q0 = bits_f32(qv[i] << 16), q1 = bits_f32(qv[i] & 0xffff0000u);
      kk = fmaf(k0, k0, fmaf(k1, k1, kk));
      qq = fmaf(q0, q0, fmaf(q1, q1, qq));
    }
    kk = sum_lanes<16>(kk);
    qq = sum_lanes<16>(qq);
    const auto most = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
    ke = over_lanes<16>(ke, most);
    qe = over_lanes<16>(qe, most);
    if (ch == 0) {
      unit[0][r] = bits_f32(0x7f000000u - (ke << 16));  // 2^(127 - e) of exponent field e
      unit[1][r] = bits_f32(0x7f000000u - (qe << 16));
      inv[0][r] = a.qk_norm ? 1.f / sqrtf(kk + kL2Eps) : 1.f;
      inv[1][r] = a.qk_norm ? 1.f / sqrtf(qq + kL2Eps) : 1.f;
    }
  }
  odd = __syncthreads_or(odd);

  const uint32_t sk = lds_addr(stage), sq = sk + kChunk * kRowB;
  if (!makes_t) {  // (the waves with less to do afterwards)
    uint8_t* img = c.keys + (id * c.khs + blockIdx.y) * kKeyImage + lane * 16;
    auto two = [](uint32_t w, float u) __attribute__((always_inline)) {  // bf16 pair times u
      return f16_pack(bits_f32(w << 16) * u, bits_f32(w & 0xffff0000u) * u);
    };
#pragma unroll
    for (int u = 0; u < 8; ++u) {  // K and Q: row block f / 4 % 4, step f % 4
      const int f = wave * 8 + u;
      const int row = 16 * ((f >> 2) & 3) + m;
      const uint32_t from = (f >= 16 ? sq : sk) + row * kRowB + (32 * (f & 3) + 4 * d) * 2;
      const float x = unit[f >> 4][row];
      const u32x2 lo = *(lds_u32x2*)(uintptr_t)from, hi = *(lds_u32x2*)(uintptr_t)(from + 32);
      st16(img + f * kFrag, u32x4{two(lo.x, x), two(lo.y, x), two(hi.x, x), two(hi.y, x)});
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {  // K^T: keys 16 (f / 2) + m, tokens of step f % 2
      const int f = wave * 4 + u;
      u32x4 w;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        // 16 lanes name 4 tokens' rows of 16 keys, a lane gets one key of the 4 (transposing)
        const int t = 32 * (f & 1) + 16 * y + 4 * d;
        const uint32_t at = sk + (t + (m >> 2)) * kRowB + (16 * (f >> 1) + 4 * (m & 3)) * 2;
        const u32x2 k4 = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)at));
        const f32x4 by = *(const f32x4*)&unit[0][t];
        w[2 * y] = f16_pack(bits_f32(k4.x << 16) * by[0], bits_f32(k4.x & 0xffff0000u) * by[1]);
        w[2 * y + 1] = f16_pack(bits_f32(k4.y << 16) * by[2], bits_f32(k4.y & 0xffff0000u) * by[3]);
      }
      st16(img + (32 + f) * kFrag, w);
    }
  }
  // without norms, keys far from 1 would put u far from the state's scale: u
  // goes in times the largest row's power of two
  float size = 1.f;
  if (!a.qk_norm) {
    // (unit: the reciprocals of the rows' sizes)
    const float x = over_lanes<64>(unit[0][lane], [](float a, float b) { return fminf(a, b); });
    size = fmaxf(1.f / x, 0x1p-30f);
  }

  // rows 16 t + m of K or Q as operands, and their products with the rows of block nt:
  // lane (m, d) has those of row 16 mt + m with rows 16 nt + 4 d + r
  auto rows_of = [&](uint32_t base, int t, u32x4 (&x)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 4; ++s) x[s] = lds_ld16(base + (16 * t + m) * kRowB + (32 * s + 8 * d) * 2);
  };
  auto products = [&](const u32x4 (&kn)[4], const u32x4 (&x)[4]) __attribute__((always_inline)) {
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s) sum = mfma(kn[s], x[s], sum);
    return sum;
  };
  for (int32_t o0 = 0; o0 < a.group; o0 += kSlots) {
    const int32_t o = o0 + slot;
    const bool there = o < a.group;  // uniform
    if (o0 > 0) {
      g = beta = 0.f;
      if (there && lane < len) load_gates(a, t0 + lane, kh * a.group + o, g, beta);
    }
    const float grow = sum_lanes<64>(fmaxf(g, 0.f));
    bool walk = odd || !(grow <= 2.f) ||
                __builtin_amdgcn_ballot_w64(!(g <= 2.f) || !(fabsf(beta) < 0x1p20f)) != 0;
    double gsum = g < (float)kLeastDecay ? kLeastDecay : (double)g;
    gsum += lanes_below<0x111>(gsum);
    gsum += lanes_below<0x112>(gsum);
    gsum += lanes_below<0x114>(gsum);
    gsum += lanes_below<0x118>(gsum);
    gsum += lanes_below<0x142, 0xa>(gsum);  // the row before's last, in rows 1 and 3
    gsum += lanes_below<0x143, 0xc>(gsum);  // lane 31's, in rows 2 and 3
    if (o0 > 0) __syncthreads();  // the last heads' readers are done
    if (!makes_t) {
      run[slot][lane] = gsum;
#pragma unroll
      for (int mt = 1; mt < 4; ++mt) {
        const double x = lane_at(gsum, 16 * mt) - gsum;
        if (lane < 16 * mt) since[slot][8 * mt * (mt - 1) + lane] = exp_of(x);
      }
    }
    __syncthreads();
    if (!there) continue;
    // e^(G_i - G_j), i = 16 mt + m, j = 16 nt + 4 d + r; below the diagonal
    // block by way of the row block's first token
    auto decays = [&](int mt, int nt, double gi, float from) __attribute__((always_inline)) {
      f32x4 e;
      if (nt < mt) {
        e = *(const f32x4*)&since[slot][8 * mt * (mt - 1) + 16 * nt + 4 * d];
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] *= from;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          e[r] = exp_of(4 * d + r <= m ? gi - run[slot][16 * nt + 4 * d + r] : 0.);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) e[r] *= inv[0][16 * nt + 4 * d + r];
      return e;
    };
    uint8_t* img = c.heads + ((id * c.khs + blockIdx.y) * a.group + o) * head_image(DELTA);
    float* fac = (float*)(img + head_image(DELTA) - kFactors);
    float largest = 0.f;  // of the operands written below
    if (!makes_t) {
      const double all = lane_at(gsum, 63);
      const float rk = inv[0][lane] / unit[0][lane], rq = inv[1][lane] / unit[1][lane];
      const float head = exp_of(gsum), strong = DELTA ? beta * size : size;
      fac[kFacX + lane] = head * rk * strong;
      const float most =
          over_lanes<64>(fabsf(strong), [](float x, float y) { return fmaxf(x, y); });
      const float by = (DELTA ? kTScale : 1.f) * kPScale;  // of P u
      fac[kFacU + lane] = exp_of(all - gsum) * rk / (DELTA ? size * kTScale : size);
      fac[kFacG + lane] = head * by;
      fac[kFacO + lane] = a.scale * rq / by;
      fac[kFacV + lane] = strong;
      fac[kFacLog + lane] = (float)(gsum * 1.4426950408889634074);
      uint8_t* pimg = img + (DELTA ? kTParts * kLower * kFrag : 0) + lane * 16;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        u32x4 qm[4];
        rows_of(sq, mt, qm);
        const double gi = run[slot][16 * mt + m];
        const float from = exp_of(gi - run[slot][16 * mt]), qi = unit[1][16 * mt + m] / size * kPScale;
        float p[8];
#pragma unroll
        for (int nt = 0; nt <= mt; ++nt) {
          u32x4 kn[4];
          rows_of(sk, nt, kn);
          const f32x4 qk = products(kn, qm), e = decays(mt, nt, gi, from);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[4 * (nt & 1) + r] = nt < mt || 4 * d + r <= m ? qi * e[r] * qk[r] : 0.f;
            if (!(nt & 1)) p[4 + r] = 0.f;
          }
          if ((nt & 1) || nt == mt) {
#pragma unroll
            for (int r = 0; r < 8; r += 2) largest = most_of(largest, p[r], p[r + 1]);
            const u32x4 high = cut(p);
            st16(pimg + lower(mt, nt >> 1) * kFrag, high);
            st16(pimg + (kLower + lower(mt, nt >> 1)) * kFrag, upper(p));
          }
          __builtin_amdgcn_sched_barrier(0);  // (registers: one block's reads at a time)
        }
      }
      walk |= __builtin_amdgcn_ballot_w64(!(largest < kMostPart)) != 0;
      if (lane == 0) {
        fac[kFacAll] = exp_of(all);
        fac[kFacMax] = most;
        ((int32_t*)fac)[kFacWalk] = walk;
        if (!DELTA) ((int32_t*)fac)[kFacWalk + 1] = 0;
      }
    } else if (DELTA) {
      const uint32_t blk = lds_addr(blocks[slot]);
      // element (row i, 4 columns from 4 x) of block n
      auto block4 = [&](int n, int i, int x) __attribute__((always_inline)) {
        return blk + (uint32_t)(n * kFrag + i * 64 + ((x ^ ((i >> 2) & 3)) << 4));
      };
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        u32x4 km[4];
        rows_of(sk, mt, km);
        const double gi = run[slot][16 * mt + m];
        const float from = exp_of(gi - run[slot][16 * mt]);
        const float ki = inv[0][16 * mt + m] * __shfl(beta, 16 * mt + m);
#pragma unroll
        for (int nt = 0; nt <= mt; ++nt) {
          u32x4 kn[4];
          if (nt < mt) rows_of(sk, nt, kn);
          f32x4 av = nt < mt ? products(kn, km) : products(km, km);
          const f32x4 e = decays(mt, nt, gi, from);
#pragma unroll
          for (int r = 0; r < 4; ++r) av[r] = nt < mt || 4 * d + r < m ? ki * e[r] * av[r] : 0.f;
          lds_st16(block4(mt * (mt + 1) / 2 + nt, m, d), __builtin_bit_cast(u32x4, av));
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      wave_sync();
      {  // the diagonal blocks' inverses: lane (m, d) has column m of block d's
        float t[16];
        const int n = d * (d + 1) / 2 + d;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float acc = i == m ? 1.f : 0.f;
#pragma unroll
          for (int x = 0; x < (i + 3) / 4; ++x) {
            const f32x4 av = lds_ldf4(block4(n, i, x));
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (4 * x + r < i) acc = fmaf(-av[r], t[4 * x + r], acc);
          }
          t[i] = acc;
        }
        wave_sync();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          *(lds_f32*)(uintptr_t)(block4(n, i, m >> 2) + (m & 3) * 4) = t[i];
        wave_sync();
      }
      f32x4 tb[kBlocks];  // T's blocks as results: lane has rows 4 d + r, column m
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const int diag = mt * (mt + 1) / 2 + mt;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          tb[diag][r] = *(lds_f32*)(uintptr_t)(block4(diag, 4 * d + r, m >> 2) + (m & 3) * 4);
        const f32x4 left = lds_ldf4(block4(diag, m, d));
#pragma unroll
        for (int nt = 0; nt < mt; ++nt) {  // -T_mm sum_x A_mx T_xn
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int x = nt; x < mt; ++x) {
            const f32x4 av = lds_ldf4(block4(mt * (mt + 1) / 2 + x, m, d));
#pragma unroll
            for (int s = 0; s < 4; ++s)
              acc = __builtin_amdgcn_mfma_f32_16x16x4f32(av[s], tb[x * (x + 1) / 2 + nt][s], acc, 0,
                                                         0, 0);
          }
          f32x4 res = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < 4; ++s)
            res = __builtin_amdgcn_mfma_f32_16x16x4f32(-left[s], acc[s], res, 0, 0, 0);
          tb[mt * (mt + 1) / 2 + nt] = res;
        }
      }
      wave_sync();
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) {
        largest = most_of(most_of(largest, tb[n][0], tb[n][1]), tb[n][2], tb[n][3]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          *(lds_f32*)(uintptr_t)(block4(n, 4 * d + r, m >> 2) + (m & 3) * 4) = tb[n][r];
      }
      wave_sync();
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int s = 0; s <= mt >> 1; ++s) {
          float x[8];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int nt = 2 * s + y;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (nt <= mt) v = lds_ldf4(block4(mt * (mt + 1) / 2 + nt, m, d));
#pragma unroll
            for (int r = 0; r < 4; ++r) x[4 * y + r] = kTScale * v[r];
          }
#pragma unroll
          for (int part = 0; part < kTParts; ++part) {
            const u32x4 w = part + 1 < kTParts ? cut(x) : upper(x);
            st16(img + lane * 16 + (part * kLower + lower(mt, s)) * kFrag, w);
          }
        }
      const bool out_of_range = __builtin_amdgcn_ballot_w64(!(largest < kMostPart / kTScale)) != 0;
      if (lane == 0) ((int32_t*)fac)[kFacWalk + 1] = out_of_range;
    }
  }
}

// Instruction classes of __builtin_amdgcn_sched_group_barrier.
constexpr int kSchedValu = 0x002, kSchedMfma = 0x008, kSchedDsRead = 0x100;

// 16 bytes per lane from base + voff into LDS at lds + 16 * lane, issued from
// inline assembly so that the compiler neither waits for it nor moves LDS
// accesses across it; the waits are explicit. M0 holds the destination.
__device__ __forceinline__ void dma16(const uint8_t* base, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(base)
               : "memory");
}
// every load and store of this wave is done, and every wave of the workgroup
// has come here
__device__ __forceinline__ void arrive_all() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// What a workgroup of linear_chunk_kernel walks: whole sequences (from slot to
// slot), or segments of them in two passes. A segment's final state is affine in
// its first one, S -> S M + B: kEnds computes B (a walk from zeros, or from the
// slot for a sequence's first segment) and M (a walk of 128 more rows from the
// identity with v = 0; without the delta rule M is a factor),
// linear_join_kernel the segments' first states from them, and kRows walks
// again from those and writes the outputs.
enum { kWhole = 0, kEnds = 1, kRows = 2 };

// One workgroup of WAVES waves per 16 WAVES value dims of a (head, sequence or
// segment); wave w holds the state of 16 of them in registers, as results of
// 16x16x32 (lane (n, d): value dim n, keys 16 x + 4 d + r), which are also the B
// operands of K S0^T and Q S0^T. The images of a chunk go straight into LDS,
// shared by the waves, while the chunk before it is computed: two buffers, one
// barrier a chunk. Bound by instruction issue: with 4 waves a chunk takes 3.6 us
// (8 x 4096 tokens, 8 heads, whole on 128 CUs: 230 us), a wave alone on its SIMD; with
// 8 waves 5.6 (32768 tokens in segments of 16 chunks: 95 us) for 682 vector, 132 matrix
// and 95 LDS instructions a wave, with the output norm 7.1 and 972 vector, with 16
// waves (no outputs, 128 value dims and 128 rows of M) 6.2.
template <int WAVES, bool DELTA, int MODE, bool NORM = false>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void linear_chunk_kernel(LinArgs a, ChunkArgs c) {
  constexpr bool kOut = MODE != kEnds;
  static_assert(!NORM || (WAVES == 8 && kOut), "the norm is taken over a head's dims");
  // With 4 waves per SIMD these hide each other's waits in 128 registers; with
  // fewer, operands are read a step ahead.
  constexpr bool kAhead = WAVES < 16;
  // a buffer: K, K^T, T, then Q and P, then the factors (offsets from the low
  // part's base, or from the high part's for what follows it)
  constexpr int kK = 0, kKt = 16 * kFrag, kQ = 32 * kFrag;
  constexpr int kLow = (kOut ? 48 : 32) * kFrag;
  constexpr int kT = 0, kP = kT + (DELTA ? kTParts * kLower * kFrag : 0);
  constexpr int kFac = kP + (kOut ? kPParts * kLower * kFrag : 0);
  constexpr int kBuffer = kLow + kFac + kFactors;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kBuffer];
  uint32_t l0 = lds_addr(lds), l1 = l0 + kBuffer;  // this chunk's buffer, and the next one's
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, d = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroups are dealt to the 8 XCDs in turn. The value heads of a key head
  // read the same K, Q and K^T: they go to one XCD, whose L2 reads them once (8
  // x 4096 tokens: 2 to 3 % less time than one XCD a head).
  const uint32_t members = (uint32_t)(a.group * c.parts), lot = blockIdx.x / kXcds;
  const uint32_t pair = lot / members * kXcds + blockIdx.x % kXcds;  // (key head, row of the launch)
  const uint32_t member = lot % members, khl = pair % (uint32_t)c.khs;
  const int32_t y = (int32_t)(pair / (uint32_t)c.khs);  // sequence, or segment
  if (y >= c.rows) return;                              // uniform
  const int32_t part = (int32_t)(member % (uint32_t)c.parts);
  const int32_t o = (int32_t)(khl * a.group + member / c.parts);  // head of the launch
  const int32_t h = c.kh0 * a.group + o, kh = h / a.group;
  // kEnds: the waves behind the value dims' have the rows of M
  const int at_dim = part * 16 * WAVES + 16 * wave;
  const bool ident = MODE == kEnds && at_dim >= kDim;
  const int d0 = at_dim - (ident ? kDim : 0);  // the wave's value dims
  const bool first = o == 0 && part == 0 && c.kh0 == 0 && tid == 0;
  int32_t b = y;
  int64_t q0 = 0, q1 = 0, s0 = 0;  // the sequence's rows; this workgroup's first
  if (MODE != kWhole) {
    b = tile_sequence(a.cu, a.n, a.tokens, y, c.seg, q0, q1, s0);
  } else {
    s0 = q0 = ld_const(a.cu + b);
    q1 = ld_const(a.cu + b + 1);
    if (!offsets_ok(a.cu, a.n, a.tokens))
      b = kBadOffsets;
    else if (q0 == q1)
      b = kNoTile;
  }
  if (MODE != kEnds && first && y == 0 && b == kBadOffsets) raise_err(a.err, MKV_DEVERR_TABLE);
  if (b < 0) return;  // uniform
  const bool at_start = s0 == q0;
  const int64_t s1 = MODE != kWhole && s0 + c.seg < q1 ? s0 + c.seg : q1;
  const bool last = s1 == q1;
  if (MODE == kEnds && last) return;  // uniform: not asked for
  const int32_t slot = ld_const(a.slots + b);  // (its load runs with the images')
  const int64_t out_row = (int64_t)a.hv * (kDim * 2);
  uint8_t* outp = a.out + h * (kDim * 2) + (d0 + n) * 2;
  const int32_t chunks = (int32_t)((s1 - s0 + kChunk - 1) / kChunk);
  const int64_t id0 = (q0 >> 6) + b + ((s0 - q0) >> 6);
  const uint8_t* kimg = c.keys + (id0 * c.khs + (kh - c.kh0)) * kKeyImage;
  const uint8_t* himg = c.heads + (id0 * c.khs * a.group + o) * head_image(DELTA);
  const int64_t knext = (int64_t)c.khs * kKeyImage;
  const int64_t hnext = (int64_t)c.khs * a.group * head_image(DELTA);

  // A wave's loads of a chunk's images, in kLoads pieces of a few each: issued in
  // one go they would hold the wave up until the address unit has taken them.
  constexpr int kKeys = kLow / kFrag, kTs = (DELTA ? kTParts * kLower : 0);
  constexpr int kFs = kFactors / kFrag, kPs = (kOut ? kPParts * kLower : 0) + kFs;  // P, factors
  constexpr int kAll = kKeys + kTs + kPs, kEach = (kAll + WAVES - 1) / WAVES, kLoads = 3;
  auto load_images = [&](int32_t ci, uint32_t to, int piece) __attribute__((always_inline)) {
    const uint8_t* kp = kimg + ci * knext;
    const uint8_t* hp = himg + ci * hnext;
#pragma unroll
    for (int f = piece * kEach / kLoads; f < (piece + 1) * kEach / kLoads; ++f) {
      const int i = f * WAVES + wave;
      if (f * WAVES + WAVES <= kKeys || i < kKeys) {  // images lie as K, Q, K^T
        const int from = i < 16 ? i : i < 32 ? i + 16 : i - 16;
        dma16(kp + from * kFrag, lane * 16, to + i * kFrag);
      } else if (i < kAll) {
        const int j = i - kKeys, from = kOut || j < kTs ? j : j + kPParts * kLower;
        dma16(hp + from * kFrag, lane * 16, to + kLow + j * kFrag);
      }
    }
  };
  // A chunk's rows of v and out through buffer descriptors that end with the
  // sequence: loads past it give zeros, stores past it are dropped, and the 16
  // rows of a lane need one address register.
  auto rows_of = [&](const uint8_t* base, int64_t stride, int32_t ci) __attribute__((always_inline)) {
    const int64_t t0 = s0 + (int64_t)ci * kChunk;
    const int32_t len = (int32_t)(s1 - t0 < kChunk ? s1 - t0 : kChunk);
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(base + t0 * stride + h * (kDim * 2)), (short)0,
        (int)((len - 1) * (int32_t)stride + kDim * 2), 0x00020000);
  };
  const int32_t vs = (int32_t)a.v_stride, os = (int32_t)out_row;
  // Memory has a token's value dims next to each other, a lane two tokens of one
  // dim: lanes in pairs move two dims each, the even one of the first token and
  // the odd one of the second, and swap halves.
  const int odd = n & 1;
  const uint32_t vat = (uint32_t)((4 * d + odd) * vs + (d0 + n - odd) * 2);
  const uint32_t oat = (uint32_t)((4 * d + odd) * os + (d0 + n - odd) * 2);
  const uint32_t halves = odd ? 0x03020706u : 0x05040100u;
  auto swap_pair = [&](uint32_t w) __attribute__((always_inline)) {
    const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xb1, 0xf, 0xf, true);
    return __builtin_amdgcn_perm(other, w, halves);
  };
  // bf16 of this lane's value dim, tokens 16 x + 4 d + (2 y, 2 y + 1) at 2 x + y; of
  // the next chunk as they come
  uint32_t v[8], vnext[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) vnext[i] = 0;
  auto load_v = [&](int32_t ci) __attribute__((always_inline)) {
    if (MODE == kEnds && ident) return;  // uniform
    const __amdgpu_buffer_rsrc_t rows = rows_of(a.v, a.v_stride, ci);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      vnext[i] =
          __builtin_amdgcn_raw_buffer_load_b32(rows, vat, (16 * (i >> 1) + 2 * (i & 1)) * vs, 0);
  };

  const int64_t row0 = (int64_t)(d0 + n) * kDim + 4 * d;  // this lane's first key of its value dim
  float* st = a.state + ((int64_t)slot * a.hv + h) * kStateHead + row0;
  const int64_t segment = ((int64_t)y * c.khs * a.group + o) * kStateHead;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) load_images(0, l0, i);
  load_v(0);
  if (slot < 0 || slot >= a.pool_slots) {  // uniform
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (loads into LDS do not outlive it)
    if (!kOut) return;
    if (first && at_start) raise_err(a.err, MKV_DEVERR_STATE_SLOT);
    for (int64_t t = s0 + d; t < s1; t += 4) *(uint16_t*)(outp + t * out_row) = 0;
    return;
  }
  f32x4 s[8];
  if (MODE == kEnds && (ident || !at_start)) {
#pragma unroll
    for (int x = 0; x < 8; ++x)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[x][r] = ident && 16 * x + 4 * d + r == d0 + n ? 1.f : 0.f;
  } else {
    const float* from = MODE == kRows && !(at_start && last) ? c.ends + segment + row0 : st;
#pragma unroll
    for (int x = 0; x < 8; ++x)
      s[x] = __builtin_bit_cast(f32x4, ld16((const uint8_t*)(from + 16 * x)));
  }
  float whole = 1.f;  // kEnds without the delta rule: the segment's decay

  // The state times f, of each value dim its own (a lane has one, 4 lanes share it).
  float f = 1.f, inv_f = 1.f;
  auto over_dim = [&](float x) __attribute__((always_inline)) {
    return over_rows(x, [](float y, float z) { return fmaxf(y, z); });
  };

  uint32_t ob[8];  // O in bf16, as v
  auto store_o = [&](int32_t ci) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t rows = rows_of(a.out, out_row, ci);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      __builtin_amdgcn_raw_buffer_store_b32(swap_pair(ob[i]), rows, oat,
                                            (16 * (i >> 1) + 2 * (i & 1)) * os, 0);
  };
  // The output norm. Each wave leaves its dims' sums of squares of a chunk's tokens in
  // LDS; behind the next chunk's barrier they are added up, and the outputs, still in
  // registers, are normed and stored.
  __shared__ __attribute__((aligned(16))) float sums[NORM ? 2 : 1][NORM ? kChunk : 1][8];
  __shared__ __attribute__((aligned(16))) float rms[NORM ? WAVES : 1][kChunk];
  f32x4 held_o[4];   // outputs of the chunk before: tokens 16 x + 4 d + r
  uint32_t held_z[8];  // their z, as v
  const float weight = NORM ? weight_at(a.w, a.w_bf16, d0 + n) : 0.f;
  auto load_z = [&](int32_t ci) __attribute__((always_inline)) {
    if (a.z_stride <= kMostStride) {  // uniform
      const int32_t zs = (int32_t)a.z_stride;
      const uint32_t zat = (uint32_t)((4 * d + odd) * zs + (d0 + n - odd) * 2);
      const __amdgpu_buffer_rsrc_t rows = rows_of(a.z, a.z_stride, ci);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        held_z[i] =
            __builtin_amdgcn_raw_buffer_load_b32(rows, zat, (16 * (i >> 1) + 2 * (i & 1)) * zs, 0);
    } else {
      const int64_t t0 = s0 + (int64_t)ci * kChunk + 4 * d + odd;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t t = t0 + 16 * (i >> 1) + 2 * (i & 1);
        held_z[i] = 0u;
        if (t < s1)
          held_z[i] = *(const uint32_t*)(a.z + t * a.z_stride + (h * kDim + d0 + n - odd) * 2);
      }
    }
  };
  auto leave_sums = [&](int32_t ci) __attribute__((always_inline)) {
    // sums over the 16 dims of a row of lanes; lane (n, d) comes to have token 16 (n / 4)
    // + 4 d + n % 4: half the tokens are given away for each of the first two bits of n
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = held_o[i >> 2][i & 3] * held_o[i >> 2][i & 3];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float keep = n & 1 ? x[2 * i + 1] : x[2 * i], give = n & 1 ? x[2 * i] : x[2 * i + 1];
      x[i] = keep + lane_of<0xb1>(give);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float keep = n & 2 ? x[2 * i + 1] : x[2 * i], give = n & 2 ? x[2 * i] : x[2 * i + 1];
      x[i] = keep + lane_of<0x4e>(give);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] += lane_of<0x128>(x[i]);  // rotations of a row by 8 and 4 lanes
      x[i] += lane_of<0x124>(x[i]);
    }
    const float y01 = n & 4 ? x[1] : x[0], y23 = n & 4 ? x[3] : x[2];
    sums[ci & 1][16 * (n >> 2) + 4 * d + (n & 3)][wave] = n & 8 ? y23 : y01;
  };
  auto store_normed = [&](int32_t ci) __attribute__((always_inline)) {
    const f32x4 lo = *(const f32x4*)&sums[ci & 1][lane][0], hi = *(const f32x4*)&sums[ci & 1][lane][4];
    const float q = ((lo[0] + lo[1]) + (lo[2] + lo[3])) + ((hi[0] + hi[1]) + (hi[2] + hi[3]));
    rms[wave][lane] = 1.f / sqrtf(q * (1.f / kDim) + a.eps);
    wave_sync();
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      const f32x4 by = *(const f32x4*)&rms[wave][16 * mt + 4 * d];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t z = swap_pair(held_z[2 * mt + y]);
        ob[2 * mt + y] =
            pack_bf16(held_o[mt][2 * y] * by[2 * y] * weight * silu_bf16(bits_f32(z << 16)),
                      held_o[mt][2 * y + 1] * by[2 * y + 1] * weight *
                          silu_bf16(bits_f32(z & 0xffff0000u)));
      }
    }
    wave_sync();  // (rms is read)
    store_o(ci);
  };
  bool stored = true;
  for (int32_t ci = 0; ci < chunks; ++ci) {
    const int64_t t0 = s0 + (int64_t)ci * kChunk;
    const int32_t len = (int32_t)(s1 - t0 < kChunk ? s1 - t0 : kChunk);
    arrive_all();  // the chunk's images and v are there; the other buffer is read
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = swap_pair(vnext[i]);
      asm volatile("" : "+v"(v[i]));
    }
    auto value = [&](int i) __attribute__((always_inline)) {
      return bits_f32(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
    };
    if (NORM && ci > 0) store_normed(ci - 1);
    const bool more = ci + 1 < chunks;
    // lane bases of the buffer's two parts: operands lie at constants from them
    uint32_t low = l0 + lane * 16, high = l0 + kLow + lane * 16;
    asm volatile("" : "+v"(low), "+v"(high));
    uint32_t fac = l0 + kLow + kFac + d * 16;
    asm volatile("" : "+v"(fac));
    auto frag = [&](int at) __attribute__((always_inline)) { return lds_ld16(low + at); };
    auto later = [&](int at) __attribute__((always_inline)) { return lds_ld16(high + at); };
    // X = K S0^T, Y = Q S0^T. Operand reads run a step ahead of their use, and
    // the vector unit cuts the next step's state while the matrix cores run.
    f32x4 xa[4], ya[4];
    constexpr int kSets = kAhead ? 2 : 1;
    u32x4 kf[kSets][4], qf[kSets][4], sp[kSets][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) xa[i] = ya[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto read_kq = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        if (DELTA) kf[ks % kSets][mt] = frag(kK + (4 * mt + ks) * kFrag);
        if (kOut) qf[ks % kSets][mt] = frag(kQ + (4 * mt + ks) * kFrag);
      }
    };
    auto cut_state = [&](int ks) __attribute__((always_inline)) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = s[2 * ks + (j >> 2)][j & 3];
      sp[ks % kSets][0] = cut(x);
      sp[ks % kSets][1] = upper(x);
    };
    f32x4 cf[4], bf[4], ef[4];
    u32x4 tq[2][4];  // T's parts of two row blocks: (0, 1; step 0), (2, 3; 0), (2, 3; 1)
    auto read_t = [&](int to, int mt0, int ks) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          tq[to][2 * i + p] = later(kT + (p * kLower + lower(mt0 + i, ks)) * kFrag);
    };
    const float decay = *(lds_f32*)(uintptr_t)(l0 + kLow + kFac + kFacAll * 4);
    const float strong = *(lds_f32*)(uintptr_t)(l0 + kLow + kFac + kFacMax * 4);
    if (kAhead && (DELTA || kOut)) read_kq(0);
    // The dim's scale: by its state's largest element, or by its values' where these
    // are to make its new state or would not fit.
    float coarse = 0.f;  // u below it is too coarse (0: none)
    float state_size = 0.f;
    uint32_t least = 0;  // values (as bf16 bits) whose u may be below that
    auto value_quad = [&](int mt) __attribute__((always_inline)) {  // of 4 tokens in a row
      // (bf16 without its sign is ordered as an integer)
      const u16x2 x = __builtin_elementwise_max(__builtin_bit_cast(u16x2, v[2 * mt] & 0x7fff7fffu),
                                                __builtin_bit_cast(u16x2, v[2 * mt + 1] & 0x7fff7fffu));
      return (uint32_t)max(x.x, x.y);
    };
    bool large = false;  // a dim of the wave does not fit fp16
    bool small = false;  // there are such values
    {
      float held = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        held = most_of(most_of(held, s[i][0], s[i][1]), s[i][2], s[i][3]);
      const uint32_t most = max(max(value_quad(0), value_quad(1)), max(value_quad(2), value_quad(3)));
      held = over_dim(held);
      float dim = over_dim(bits_f32(most << 16)) * (strong * f);
      const bool fresh = held * decay < kLittle * dim;
      const bool by_value = fresh || !(dim < kHighValue);
      const float x = by_value ? dim : held;
      const bool out = !(x < (by_value ? kHighValue : kHighState)) ||
                       (x < (by_value ? kLowValue : kLowState) && x > 0.f);
      if (__builtin_amdgcn_ballot_w64(out) != 0) {
        float to = bits_f32(0x7f000000u + ((by_value ? kNearValue : kNearState) << 23) -
                            (f32_bits(x) & 0x7f800000u));
        if (!out || !(x > 0x1p-110f && x < 0x1p120f && f * to > 0x1p-100f && f * to < 0x1p100f))
          to = 1.f;
        f *= to;
        inv_f = 1.f / f;
        held *= to;
        dim *= to;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[i][r] *= to;
      }
      large = __builtin_amdgcn_ballot_w64(!(held < kMostState)) != 0;
      // (M's rows are taken of what was before the segment: what a chunk's largest leave
      // in them, 2^-28 of it, is of no matter)
      if (!ident && fresh)
        coarse = dim < kLowValue ? 3e38f : kLeastQuad * (DELTA ? dim + 4.f * held : dim);
      else if (!ident && decay < kLeastState && dim < kLeastValue * held && dim > 0.f)
        coarse = 3e38f;
      if (coarse > 0.f) least = f32_bits(coarse * __builtin_amdgcn_rcpf(strong * f)) >> 16;
      state_size = held;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) small |= value_quad(mt) < least && value_quad(mt) != 0;
    }
    if (kAhead && (DELTA || kOut)) cut_state(0);
    if (more) load_v(ci + 1);
    if (kAhead) __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (!kAhead && (DELTA || kOut)) {
        read_kq(ks);
        cut_state(ks);
      } else if (ks < 3) {
        if (DELTA || kOut) {
          read_kq(ks + 1);
          cut_state(ks + 1);
        }
      }
      if (kAhead && DELTA && ks == 3) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          cf[mt] = lds_ldf4(fac + (kFacX + 16 * mt) * 4);
          bf[mt] = lds_ldf4(fac + (kFacV + 16 * mt) * 4);
        }
        read_t(0, 0, 0);
      }
      if (DELTA || kOut) {
#pragma unroll
        for (int p = 1; p >= 0; --p) {
          if (DELTA)
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) xa[mt] = mfma16(kf[ks % kSets][mt], sp[ks % kSets][p], xa[mt]);
          if (kOut)
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) ya[mt] = mfma16(qf[ks % kSets][mt], sp[ks % kSets][p], ya[mt]);
        }
        if (kAhead && ks < 3) {
          __builtin_amdgcn_sched_group_barrier(kSchedDsRead, (DELTA ? 4 : 0) + (kOut ? 4 : 0), 0);
#pragma unroll
          for (int i = 0; i < (DELTA ? 8 : 0) + (kOut ? 8 : 0); ++i) {
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kSchedValu, 2, 0);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (ks < kLoads && more) load_images(ci + 1, l1, ks);
    }
    __builtin_amdgcn_s_setprio(0);
    const u32x2 walks = *(lds_u32x2*)(uintptr_t)(l0 + kLow + kFac + kFacWalk * 4);
    const uint32_t walk = __builtin_amdgcn_readfirstlane(walks.x | walks.y);
    if (MODE == kEnds && !DELTA) whole *= decay;
    const uint32_t lnow = l0;
    l0 = l1;
    l1 = lnow;
    f32x4 u[4], rhs[4];
    bool big = false;  // operands past their limits, infinities and NaN
    auto check = [&](const f32x4 (&x)[4]) __attribute__((always_inline)) {
      float most = 0.f;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) most = any_of(any_of(most, x[mt][0], x[mt][1]), x[mt][2], x[mt][3]);
      big = !(most < kMostRhs);
    };
    u32x4 pf[kPParts][4], tf[8];  // operands of P and of K^T
    auto read_p = [&](int p, int ks) __attribute__((always_inline)) {
      if (!kOut) return;
#pragma unroll
      for (int mt = 2 * ks; mt < 4; ++mt) pf[p][mt] = later(kP + (p * kLower + lower(mt, ks)) * kFrag);
    };
    auto read_kt = [&](int ks, int from, int to) __attribute__((always_inline)) {
#pragma unroll
      for (int i = from; i < to; ++i) tf[i] = frag(kKt + (2 * i + ks) * kFrag);
    };
    if (DELTA) {
      if (!kAhead) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          cf[mt] = lds_ldf4(fac + (kFacX + 16 * mt) * 4);
          bf[mt] = lds_ldf4(fac + (kFacV + 16 * mt) * 4);
        }
      } else {
        read_t(1, 2, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          rhs[mt][r] = fmaf(value(4 * mt + r), bf[mt][r] * f, -cf[mt][r] * xa[mt][r]);
      check(rhs);
    } else {
      const float bf = *(lds_f32*)(uintptr_t)(lnow + kLow + kFac + kFacV * 4) * f;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int r = 0; r < 4; ++r) u[mt][r] = value(4 * mt + r) * bf;
      check(u);
    }
    u32x4 r0[2], r1[2];
    if (DELTA) {
      auto mul_t = [&](int from, int mt0, const u32x4 (&r)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 2; p >= 0; --p)  // lower x upper, upper x lower, upper x upper
#pragma unroll
          for (int i = 0; i < 2; ++i)
            u[mt0 + i] = mfma16(tq[from][2 * i + (p == 2)], r[p == 1], u[mt0 + i]);
      };
      auto cut_rhs = [&](int ks, u32x4 (&to)[2]) __attribute__((always_inline)) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = rhs[2 * ks + (j >> 2)][j & 3];
        to[0] = cut(x);
        to[1] = upper(x);
      };
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) u[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
      cut_rhs(0, r0);
      if (kAhead)
        __builtin_amdgcn_sched_barrier(0);
      else
        read_t(0, 0, 0);
      cut_rhs(1, r1);
      mul_t(0, 0, r0);
      if (!kAhead) {
        __builtin_amdgcn_sched_barrier(0);
        read_t(1, 2, 0);
      }
      mul_t(1, 2, r0);
      if (kAhead) {
#pragma unroll
        for (int i = 0; i < 12; ++i) {
          __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
          __builtin_amdgcn_sched_group_barrier(kSchedValu, 2, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      // (T's last blocks have been waited for; the others' use comes after more work)
      read_t(0, 2, 1);
    }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) ef[mt] = lds_ldf4(fac + (kFacU + 16 * mt) * 4);
    read_p(1, 0);
    if (kAhead) __builtin_amdgcn_sched_barrier(0);
    if (kOut && !NORM && !stored) store_o(ci - 1);
    stored = false;
    if (NORM) load_z(ci);
    if (DELTA) {
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          u[2 + i] = mfma16(tq[0][2 * i + (p == 2)], r1[p == 1], u[2 + i]);
    }
    // (fp16 operands: limits of u, and of u times its factors in the state)
    {
      float most = 0.f;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
        for (int r = 0; r < 4; ++r) ef[mt][r] *= u[mt][r];
        most = most_of(most_of(most, u[mt][0], u[mt][1]), u[mt][2], u[mt][3]);
        most = most_of(most_of(most, ef[mt][0], ef[mt][1]), ef[mt][2], ef[mt][3]);
      }
      big |= !(most < kMostPart);
    }
    bool by_token = walk != 0 || large || __builtin_amdgcn_ballot_w64(big) != 0;
    if (__builtin_expect(!by_token && __builtin_amdgcn_ballot_w64(small) != 0, 0)) {
      // log2 of what is left at a token of all before it, and of the state: of the largest
      // of log2 |u_j| - log2 e^G_j, and then times e^G of the token
      const float scale = DELTA ? kTScale : 1.f;
      const float limit = __builtin_amdgcn_logf(coarse * scale);
      float before = __builtin_amdgcn_logf(state_size * scale);
      int32_t quads = 0;
      bool lost = false, lost_end = false;  // (the latter of a sequence's last 1 to 3 tokens)
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const f32x4 gl = lds_ldf4(fac + (kFacLog + 16 * mt) * 4);
        float own = -3e38f, quad = -3e38f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = __builtin_amdgcn_logf(fabsf(u[mt][r]));
          quad = fmaxf(quad, x);
          own = fmaxf(own, x - gl[r]);
        }
        float left = before;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float other = __shfl(own, n + 16 * k);
          left = k < d ? fmaxf(left, other) : left;
          before = fmaxf(before, other);
        }
        if (value_quad(mt) < least && value_quad(mt) != 0) {
          const bool gone = fmaxf(quad, left + gl[0]) < limit;
          if (16 * mt + 4 * d + 4 <= len) {
            ++quads;
            lost |= gone;
          } else {
            lost_end |= gone;
          }
        }
      }
      quads = over_rows(quads, [](int32_t y, int32_t z) { return y + z; });
      lost |= quads >= kManyQuads;
      // (few tokens are small by chance; not in half of the dims)
      by_token = __builtin_amdgcn_ballot_w64(lost) != 0 ||
                 __builtin_popcountll(__builtin_amdgcn_ballot_w64(lost_end)) >= 8;
    }
    if (__builtin_expect(by_token, 0)) {
      // token by token: sums over keys in the lane's registers and the 4 lanes of its value
      // dim. Lane i has token i's gates, and the next token's rows load beside this one's
      // sums: 0.7 us a token, 1.3 with all of it in line.
      auto over_keys = [&](float x) __attribute__((always_inline)) {
        return over_rows(x, [](float y, float z) { return y + z; });
      };
      float g = 0.f, beta = 0.f;
      if (lane < len) load_gates(a, t0 + lane, h, g, beta);
      const uint32_t decays = f32_bits(expf(g)), betas = f32_bits(beta);
      u32x2 kw[8], qw[8];
      float vw = 0.f;
      auto fetch = [&](int32_t t) __attribute__((always_inline)) {
        const int64_t token = t0 + t;
        const uint8_t* kp = a.k + token * a.k_stride + kh * (kDim * 2) + d * 8;
        const uint8_t* qp = a.q + token * a.q_stride + kh * (kDim * 2) + d * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          kw[i] = *(const u32x2*)(kp + 32 * i);
          if (kOut) qw[i] = *(const u32x2*)(qp + 32 * i);
        }
        if (!ident) vw = bf16_at(a.v + token * a.v_stride + (h * kDim + d0 + n) * 2);
      };
      fetch(0);
#pragma unroll 1
      for (int32_t t = 0; t < len; ++t) {
        float kx[8][4], qx[8][4], kk = 0.f, qq = 0.f, kq = 0.f, x = 0.f, y = 0.f;
        const float vt = f * vw;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          unpack4(kw[i], kx[i]);
          if (kOut) unpack4(qw[i], qx[i]);
        }
        if (t + 1 < len) fetch(t + 1);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            kk = fmaf(kx[i][r], kx[i][r], kk);
            x = fmaf(s[i][r], kx[i][r], x);
            if (kOut) {
              qq = fmaf(qx[i][r], qx[i][r], qq);
              kq = fmaf(kx[i][r], qx[i][r], kq);
              y = fmaf(s[i][r], qx[i][r], y);
            }
          }
        float rk = 1.f, rq = 1.f;
        if (a.qk_norm) {
          rk = 1.f / sqrtf(over_keys(kk) + kL2Eps);
          if (kOut) rq = 1.f / sqrtf(over_keys(qq) + kL2Eps);
        }
        const float e = bits_f32(__builtin_amdgcn_readlane(decays, t));
        const float b = bits_f32(__builtin_amdgcn_readlane(betas, t));
        const float u = DELTA ? b * (vt - e * rk * over_keys(x)) : vt;
        if (kOut) {
          const float out = a.scale * inv_f * (e * rq * over_keys(y) + u * (over_keys(kq) * rk * rq));
          if (NORM) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (16 * (i >> 2) + 4 * d + (i & 3) == t) held_o[i >> 2][i & 3] = out;
          } else if (d == 0) {
            *(uint16_t*)(outp + (t0 + t) * out_row) = f32_to_bf16_rne(out);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[i][r] = fmaf(u * rk, kx[i][r], e * s[i][r]);
      }
      if (NORM) leave_sums(ci);
      stored = true;
      continue;
    }
    // S = e^G S0 + (e^(G_63 - G) u) k^T; O = e^G Y + P U
    f32x4 eg[4], of[4];
    if (kOut) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) eg[mt] = lds_ldf4(fac + (kFacG + 16 * mt) * 4);
    }
    if (kAhead) read_kt(0, 0, 8);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = ef[2 * ks + (j >> 2)][j & 3];
      u32x4 w[2];
      w[0] = cut(x);
      w[1] = upper(x);
      if (ks == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[i][r] *= decay;
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      // the state's products while the vector unit rounds u and scales Y for the output's
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = u[2 * ks + (j >> 2)][j & 3];
      const u32x4 uh = cut(x), ul = upper(x);
      if (kOut && ks == 0) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int r = 0; r < 4; ++r) ya[mt][r] *= eg[mt][r];
      }
#pragma unroll
      for (int half = 0; half < (kAhead ? 1 : 2); ++half) {
        const int from = kAhead ? 0 : 4 * half, to = kAhead ? 8 : 4 * half + 4;
        if (!kAhead) read_kt(ks, from, to);
#pragma unroll
        for (int p = 1; p >= 0; --p)
#pragma unroll
          for (int i = from; i < to; ++i) s[i] = mfma16(tf[i], w[p], s[i]);
        if (!kAhead) __builtin_amdgcn_sched_barrier(0);
      }
      if (kOut) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
          __builtin_amdgcn_sched_group_barrier(kSchedValu, 2, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(0);
      read_p(0, ks);
      if (kAhead && ks == 0) read_kt(1, 0, 8);
      if (kOut) {
#pragma unroll
        for (int p = 2; p >= 0; --p)  // lower x upper, upper x lower, upper x upper
#pragma unroll
          for (int mt = 2 * ks; mt < 4; ++mt)
            ya[mt] = mfma16(pf[p == 2][mt], p == 1 ? ul : uh, ya[mt]);
        if (ks == 0) {
          read_p(1, 1);
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) of[mt] = lds_ldf4(fac + (kFacO + 16 * mt) * 4);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (NORM) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int r = 0; r < 4; ++r) held_o[mt][r] = ya[mt][r] * (of[mt][r] * inv_f);
      leave_sums(ci);
    } else if (kOut) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int mt = i >> 1, j = 2 * (i & 1);
        ob[i] = pack_bf16(ya[mt][j] * (of[mt][j] * inv_f), ya[mt][j + 1] * (of[mt][j + 1] * inv_f));
      }
    }
  }
  if (NORM) {
    arrive_all();
    store_normed(chunks - 1);
  } else if (kOut && !stored) {
    store_o(chunks - 1);
  }
#pragma unroll
  for (int x = 0; x < 8; ++x)
#pragma unroll
    for (int r = 0; r < 4; ++r) s[x][r] *= inv_f;
  if (MODE == kEnds) {
    if (ident && at_start) return;
    if (ident) {
      // as linear_join_kernel's operands: row block x of M^T, columns 16 y; lane
      // (m, e) has row m, columns 4 e .. +3. This lane has column n of y = d0 / 16.
      float* to = c.steps + segment + (d0 / 16) * 256 + (n >> 2) * 64 + (n & 3);
#pragma unroll
      for (int x = 0; x < 8; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) to[x * 8 * 256 + (4 * d + r) * 4] = s[x][r];
    } else {
#pragma unroll
      for (int x = 0; x < 8; ++x)
        st16((uint8_t*)(c.ends + segment + row0 + 16 * x), __builtin_bit_cast(u32x4, s[x]));
      if (!DELTA && tid == 0 && part == 0)
        c.steps[(int64_t)y * c.khs * a.group + o] = whole;
    }
  } else if (last) {
#pragma unroll
    for (int x = 0; x < 8; ++x) st16((uint8_t*)(st + 16 * x), __builtin_bit_cast(u32x4, s[x]));
  }
}

// The first states of a sequence's segments, in the place of their B: one
// workgroup per 16 value dims of a (head, sequence). S -> S M + B runs in fp32
// matrix instructions (16x16x4), each wave making 32 of the 128 keys; the state
// is handed round through LDS. Without the delta rule M is a factor. Bound by the
// chain of segments: 1.85 us each (32 segments of 8 heads: 57 us), 1.0 of them the
// 64 matrix instructions of a wave.
template <bool DELTA>
__global__ __launch_bounds__(256) void linear_join_kernel(LinArgs a, ChunkArgs c) {
  __shared__ __attribute__((aligned(16))) float state[2][kDim / 4][64];  // 4-key groups x (dim, key)
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, d = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // (a head's workgroups on one XCD where heads are a multiple of 8: M once in its L2)
  const int32_t heads = c.khs * a.group, o = blockIdx.x % heads, part = blockIdx.x / heads;
  const int32_t h = c.kh0 * a.group + o, b = blockIdx.y;
  if (!offsets_ok(a.cu, a.n, a.tokens)) return;
  const int64_t q0 = ld_const(a.cu + b), q1 = ld_const(a.cu + b + 1);
  const int32_t segs = (int32_t)((q1 - q0 + c.seg - 1) / c.seg);
  const int64_t seg0 = first_tile((int32_t)q0, b, c.seg);
  const int32_t slot = ld_const(a.slots + b);
  if (segs < 2 || slot < 0 || slot >= a.pool_slots) return;  // uniform
  const int64_t next = (int64_t)c.khs * a.group * kStateHead;
  const int64_t row = (int64_t)(16 * part + n) * kDim + 4 * d + 32 * wave;  // this wave's keys
  const int64_t at = seg0 * next + (int64_t)o * kStateHead;
  float* ends = c.ends + at + row;
  const float* slot0 = a.state + ((int64_t)slot * a.hv + h) * kStateHead + row;
  f32x4 s[2], init[2];  // keys 32 wave + 16 y + 4 d + r of value dim n
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    s[y] = __builtin_bit_cast(f32x4, ld16((const uint8_t*)(ends + 16 * y)));
    init[y] = __builtin_bit_cast(f32x4, ld16((const uint8_t*)(slot0 + 16 * y)));
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) st16((uint8_t*)(ends + 16 * y), __builtin_bit_cast(u32x4, init[y]));
  // A operand rows: keys 32 wave + 16 y + n of M^T, columns 16 x + 4 d + r, 1 KiB
  // blocks in this order; they and B are read
  const float* mt = c.steps + at + 2 * wave * 8 * 256 + lane * 4;
  // two segments ahead (three sets of registers, in turn)
  f32x4 m[3][2][8], acc[3][2];
  auto read_step = [&](int32_t i, f32x4 (&mi)[2][8], f32x4 (&bi)[2]) __attribute__((always_inline)) {
    if (i + 1 >= segs) return;  // uniform; the last segment's B and M are not asked for
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      bi[y] = __builtin_bit_cast(f32x4, ld16((const uint8_t*)(ends + i * next + 16 * y)));
      if (DELTA)
#pragma unroll
        for (int x = 0; x < 8; ++x)
          mi[y][x] = __builtin_bit_cast(
              f32x4, ld16((const uint8_t*)(mt + i * next + (y * 8 + x) * 256)));
    }
  };
  auto step = [&](int32_t i, f32x4 (&mi)[2][8], f32x4 (&bi)[2], f32x4 (&m2)[2][8],
                  f32x4 (&b2)[2]) __attribute__((always_inline)) {
    // this lane's B of the segment is read: the segment's first state takes its place
#pragma unroll
    for (int y = 0; y < 2; ++y)
      st16((uint8_t*)(ends + i * next + 16 * y), __builtin_bit_cast(u32x4, s[y]));
    if (i + 1 >= segs) return;
    read_step(i + 2, m2, b2);
    f32x4 sum[2] = {bi[0], bi[1]};
    if (DELTA) {
      float* to = &state[i & 1][0][0] + (8 * wave + d) * 64 + n * 4;
#pragma unroll
      for (int y = 0; y < 2; ++y) *(f32x4*)(to + y * 4 * 64) = s[y];
      // (a barrier for LDS alone: the loads stay in flight)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const float* from = &state[i & 1][0][0] + d * 64 + n * 4;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const f32x4 k = *(const f32x4*)(from + x * 4 * 64);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            sum[y] = __builtin_amdgcn_mfma_f32_16x16x4f32(mi[y][x][r], k[r], sum[y], 0, 0, 0);
      }
    } else {
      const float f = c.steps[(seg0 + i) * c.khs * a.group + o];
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[y][r] = fmaf(f, s[y][r], sum[y][r]);
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) s[y] = sum[y];
  };
  read_step(1, m[0], acc[0]);
  read_step(2, m[1], acc[1]);
  for (int32_t i = 1; i < segs; i += 3) {
    step(i, m[0], acc[0], m[2], acc[2]);
    if (i + 1 < segs) step(i + 1, m[1], acc[1], m[0], acc[0]);
    if (i + 2 < segs) step(i + 2, m[2], acc[2], m[1], acc[1]);
  }
}

// ---------------------------------------------------------------------------
// y = x / sqrt(mean(x^2) + eps) w silu(z), a row of `dim` values at a time
// ---------------------------------------------------------------------------
struct NormArgs {
  const uint8_t *x, *z, *w;
  int64_t x_stride, z_stride;  // bytes between tokens; a token's heads follow each other
  int32_t heads, dim, w_bf16;
  float eps;
  uint8_t* out;  // [tokens, heads, dim]
  int64_t rows;  // tokens * heads
};

// 8 weights as floats
template <bool BF16>
__device__ __forceinline__ void load_weights(const uint8_t* w, int d, float (&x)[8]) {
  if (BF16) {  // (aligned to 2 bytes)
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = bf16_at(w + 2 * (d + j));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = *(const float*)(w + 4 * (d + j));
  }
}

// LANES lanes per row, 8 values (16 bytes) per lane and step. Bound by HBM: 2^20
// rows of 128 take 130 us, 6.2 TB/s over x, z and out (four rows a thread, all
// loaded before the first is used: 139); 2048 rows 2.7 us, a launch.
template <int LANES, int STEPS, bool BF16>
__global__ __launch_bounds__(kThreads) void gated_norm_kernel(NormArgs a) {
  const int lane = threadIdx.x % LANES;
  const uint32_t heads = (uint32_t)a.heads;
  float w[STEPS][8];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int d = (s * LANES + lane) * 8;
    if (d < a.dim) load_weights<BF16>(a.w, d, w[s]);
  }
  const int64_t wg = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t row = wg * (kThreads / LANES) + threadIdx.x / LANES;
  const uint32_t at = row < a.rows ? (uint32_t)row : 0;
  const uint32_t token = heads == 1 ? at : at / heads, head = at - token * heads;
  const bool there = row < a.rows;
  const int64_t off = (int64_t)head * a.dim * 2;
  const uint8_t* xp = a.x + token * a.x_stride + off;
  const uint8_t* zp = a.z + token * a.z_stride + off;
  u32x4 xv[STEPS], zv[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int d = (s * LANES + lane) * 8;
    xv[s] = zv[s] = u32x4{0u, 0u, 0u, 0u};
    if (there && d < a.dim) {
      xv[s] = ld16(xp + 2 * d);
      zv[s] = ld_nt(zp + 2 * d);
    }
  }
  float q = 0.f;
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float lo = bits_f32(xv[s][j] << 16), hi = bits_f32(xv[s][j] & 0xffff0000u);
      q = fmaf(lo, lo, q);
      q = fmaf(hi, hi, q);
    }
  q = sum_lanes<LANES>(q);
  const float r = 1.f / sqrtf(q / (float)a.dim + a.eps);
  if (!there) return;
  uint8_t* out = a.out + row * a.dim * 2;
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int d = (s * LANES + lane) * 8;
    if (d >= a.dim) continue;
    u32x4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = xv[s][j], z = zv[s][j];
      y[j] = pack_bf16(
          bits_f32(x << 16) * r * w[s][2 * j] * silu_bf16(bits_f32(z << 16)),
          bits_f32(x & 0xffff0000u) * r * w[s][2 * j + 1] * silu_bf16(bits_f32(z & 0xffff0000u)));
    }
    st16(out + 2 * d, y);
  }
}

template <int LANES, int STEPS>
void launch_norm(const NormArgs& a, hipStream_t stream) {
  constexpr int kRowsPerWg = kThreads / LANES;
  const int64_t wgs = (a.rows + kRowsPerWg - 1) / kRowsPerWg;
  constexpr int64_t kWide = 1 << 20;  // (a grid dimension has less than 2^32 threads)
  const dim3 grid((unsigned)(wgs < kWide ? wgs : kWide), (unsigned)((wgs + kWide - 1) / kWide));
  if (a.w_bf16)
    hipLaunchKernelGGL((gated_norm_kernel<LANES, STEPS, true>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((gated_norm_kernel<LANES, STEPS, false>), grid, dim3(kThreads), 0, stream,
                       a);
}

constexpr int kNormMaxDim = 4096;
constexpr int64_t kNormMaxRows = 1ll << 30;

void run_norm(const NormArgs& a, hipStream_t stream) {
  const int32_t d = a.dim;
  if (d <= 64)
    launch_norm<8, 1>(a, stream);
  else if (d <= 128)
    launch_norm<16, 1>(a, stream);
  else if (d <= 256)
    launch_norm<32, 1>(a, stream);
  else if (d <= 512)
    launch_norm<64, 1>(a, stream);
  else if (d <= 1024)
    launch_norm<64, 2>(a, stream);
  else if (d <= 2048)
    launch_norm<64, 4>(a, stream);
  else
    launch_norm<64, 8>(a, stream);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// What the two forms ask of their arguments alike; fills `a`.
int linear_args(const char* fn, void* state, int64_t pool_slots, int32_t hk, int32_t hv,
                int32_t head_dim, const int32_t* slots, int32_t n, int64_t tokens, const void* q,
                int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                const void* g, int64_t g_stride, const void* beta, int64_t beta_stride,
                int32_t gates_bf16, const float* a_log, const float* dt_bias, int32_t qk_norm,
                float scale, const void* z, int64_t z_stride, const void* w, int32_t w_bf16,
                float eps, void* out, int32_t* err, LinArgs& a) {
  MKV_REQUIRE(pool_slots >= 0 && n >= 0 && tokens >= 0 && hk > 0 && hv > 0, MKV_E_INVALID,
              "%s: bad sizes", fn);
  MKV_REQUIRE(head_dim == kDim, MKV_E_UNSUPPORTED, "%s: head_dim %d unsupported (128)", fn,
              head_dim);
  MKV_REQUIRE(hv % hk == 0 && hv <= 1024, MKV_E_UNSUPPORTED,
              "%s: %d value heads on %d key heads unsupported (a multiple, at most 1024)", fn, hv,
              hk);
  MKV_REQUIRE(n <= 65535, MKV_E_UNSUPPORTED, "%s: batch above 65535", fn);
  if (n == 0 || tokens == 0) return MKV_OK;  // (the caller launches nothing)
  MKV_REQUIRE(state && slots && q && k && v && g && out && err, MKV_E_INVALID, "%s: null pointer",
              fn);
  MKV_REQUIRE((a_log == nullptr) == (dt_bias == nullptr), MKV_E_INVALID,
              "%s: a_log and dt_bias come together", fn);
  MKV_REQUIRE((z == nullptr) == (w == nullptr), MKV_E_INVALID,
              "%s: a gate and its norm's weight come together", fn);
  const int64_t krow = (int64_t)hk * kDim * 2, vrow = (int64_t)hv * kDim * 2;
  const int64_t grow = (int64_t)hv * (gates_bf16 ? 2 : 4);
  MKV_REQUIRE(q_stride >= krow && k_stride >= krow && v_stride >= vrow && g_stride >= grow &&
                  (!beta || beta_stride >= grow) && (!z || z_stride >= vrow),
              MKV_E_INVALID, "%s: a stride is shorter than its row", fn);
  MKV_REQUIRE(aligned16(state) && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) &&
                  aligned16(z) && q_stride % 16 == 0 && k_stride % 16 == 0 && v_stride % 16 == 0 &&
                  z_stride % 16 == 0,
              MKV_E_ALIGN, "%s: state, rows and their strides must be 16-byte aligned", fn);
  const int64_t ge = gates_bf16 ? 2 : 4;
  MKV_REQUIRE((uintptr_t)g % ge == 0 && (uintptr_t)beta % ge == 0 && g_stride % ge == 0 &&
                  beta_stride % ge == 0 && aligned4(a_log) && aligned4(dt_bias) &&
                  (uintptr_t)w % (w_bf16 ? 2 : 4) == 0,
              MKV_E_ALIGN, "%s: gates and weights must be aligned to their type", fn);
  a.state = (float*)state;
  a.pool_slots = pool_slots;
  a.slots = slots;
  a.n = n;
  a.hk = hk;
  a.hv = hv;
  a.group = hv / hk;
  a.q = (const uint8_t*)q;
  a.k = (const uint8_t*)k;
  a.v = (const uint8_t*)v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.g = (const uint8_t*)g;
  a.beta = (const uint8_t*)beta;
  a.g_stride = g_stride;
  a.beta_stride = beta_stride;
  a.gates_bf16 = gates_bf16;
  a.a_log = a_log;
  a.dt_bias = dt_bias;
  a.qk_norm = qk_norm;
  a.scale = scale;
  a.z = (const uint8_t*)z;
  a.w = (const uint8_t*)w;
  a.z_stride = z_stride;
  a.w_bf16 = w_bf16;
  a.eps = eps;
  a.out = (uint8_t*)out;
  a.tokens = tokens;
  a.err = err;
  return MKV_OK;
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" int mkv_linear_attn_decode(
    void* state, int64_t pool_slots, int32_t num_k_heads, int32_t num_v_heads, int32_t head_dim,
    const int32_t* slots, int32_t batch, const void* q, int64_t q_stride, const void* k,
    int64_t k_stride, const void* v, int64_t v_stride, const void* g, int64_t g_stride,
    const void* beta, int64_t beta_stride, int32_t gates_bf16, const float* a_log,
    const float* dt_bias, int32_t qk_norm, float scale, const void* z, int64_t z_stride,
    const void* norm_weight, int32_t weight_bf16, float norm_eps, void* out, int32_t* err,
    void* stream) {
  clear_error();
  const char* fn = "mkv_linear_attn_decode";
  LinArgs a{};
  const int rc = linear_args(fn, state, pool_slots, num_k_heads, num_v_heads, head_dim, slots,
                             batch, batch, q, q_stride, k, k_stride, v, v_stride, g, g_stride,
                             beta, beta_stride, gates_bf16, a_log, dt_bias, qk_norm, scale, z,
                             z_stride, norm_weight, weight_bf16, norm_eps, out, err, a);
  if (rc != MKV_OK) return rc;
  if (batch == 0) return MKV_OK;
  const dim3 grid((unsigned)num_v_heads, (unsigned)batch);
  hipLaunchKernelGGL(linear_decode_kernel, grid, dim3(kThreads), 0, as_stream(stream), a);
  return check_launch(fn);
}

namespace mkv {
namespace {

constexpr int64_t kLeastBytes = 16;  // of a workspace, so that no call goes without one
// Images of one launch at most: more key heads, or value heads of one, are run in turn
// in the same space, which leaves CUs idle (16/64 heads, 32768 tokens, 1.2 GiB of
// images: 1723 us at once; in launches of 13 and 3 key heads 2813, of 6, 6 and 4 2010).
// One value head at least: 74 KiB for 64 tokens.
constexpr int64_t kImageBytes = 2048ll << 20;
// Up to so many tokens per sequence are walked one by one (8 heads; token by
// token, in chunks: 1 sequence of 8 tokens 15 us, 15; 32 of 8 23, 29; 64 of 8
// 37, 45; of 12 51, 44; 256 of 4 73, 121; of 8 113, 122; with the norm 2 to 12 more).
constexpr int32_t kScanTokens = 8;

constexpr double kMostThreads = 4294967296.;  // of a grid dimension, less than this
constexpr int32_t kPrepThreads = 512;

struct Prefill {
  bool chunked;
  int64_t ids;    // tiles
  int32_t waves;  // of a workgroup that writes outputs (a head's value dims take 8)
  int32_t seg;    // tokens of a segment; 0: whole sequences
  int32_t end_waves;  // of a workgroup that computes segments' ends
  int64_t segs;   // segment ids
  int32_t khs;    // key heads of a launch
  int32_t vhs;    // value heads of each: all, or some of a single one's
  int64_t key_bytes, head_bytes, end_bytes, step_bytes, total;
};

// What a pass takes (us on MI355X, fitted to 12 shapes of 1 to 32 sequences of
// 300 to 32768 tokens under all choices, 4 % off on average): so many a chunk
// where up to half the CUs have a workgroup, and where all have (normed8: by 8 waves
// with the output norm); a join so many a segment.
struct ChunkCosts {
  float rows4[2], rows8[2], normed8[2], ends8[2], ends16[2], join;
};
constexpr ChunkCosts kDeltaCosts = {{3.2f, 3.6f}, {3.9f, 5.2f}, {5.1f, 6.7f},
                                    {2.6f, 3.2f}, {4.2f, 5.7f}, 1.6f};
constexpr ChunkCosts kDecayCosts = {{2.5f, 2.6f}, {3.0f, 3.3f}, {4.2f, 4.6f},
                                    {1.6f, 2.5f}, {1.6f, 2.5f}, 0.35f};
constexpr float kPassStart = 5.5f;  // a pass's launch, its first loads and its last stores

// A pass of `wgs` workgroups of at most `chunks` chunks each, one per CU at a time.
float pass_time(const float (&cost)[2], double wgs, double chunks, int cus, double uneven = 1.) {
  const double half = cus / 2.0, load = wgs <= half ? 0. : wgs >= cus ? 1. : (wgs - half) / half;
  const double rounds = wgs * uneven <= cus ? 1. : ceil(wgs * uneven / cus);
  return (float)(kPassStart + rounds * chunks * (cost[0] + load * (cost[1] - cost[0])));
}

// Whole sequences or segments of them, and workgroups of half a head or of one,
// by those costs. The batch is taken as its longest sequence and others alike.
// (us, prep and all, 8 heads: 1 x 32768 tokens whole 1797, segments of 8 chunks
// 350, of 16 286, of 32 330; 8 x 4096 whole 275, segments of 16 chunks 242, with the
// norm 399 and 260; 32 x 1024 half heads 194, whole ones 151, segments of 8 chunks
// 249; 1 x 1024 whole 78, segments of 4 chunks 61; 6 of 80 to 3000 whole 182,
// segments of 6 chunks 106.)
void choose_walk(Prefill& p, int64_t tokens, int32_t n, int32_t longest, double heads, bool delta,
                 bool norm) {
  const ChunkCosts& c = delta ? kDeltaCosts : kDecayCosts;
  const int cus = device_cus();
  const double most = longest > 0 && longest < tokens ? longest : tokens;
  const double rest = n > 1 ? (tokens - most) / (n - 1) : 0;
  const double long_chunks = ceil(most / kChunk), rest_chunks = ceil(rest / kChunk);
  const double work = long_chunks + (n - 1) * rest_chunks;  // chunks of one head
  float best = 3e38f;
  for (int32_t waves = norm ? 8 : 4; waves <= 8; waves += 4) {
    const float (&cost)[2] = norm ? c.normed8 : waves == 4 ? c.rows4 : c.rows8;
    const double parts = 8.0 / waves, wgs = heads * parts * n;
    // (rounds of sequences of different lengths fill up: at least the longest one)
    const double each = wgs <= cus ? long_chunks : fmax(long_chunks, work * heads * parts / cus);
    const float t = pass_time(cost, wgs <= cus ? wgs : cus, each, cus);
    if (t < best) {
      best = t;
      p.waves = waves;
      p.seg = 0;
    }
  }
  for (int32_t len = 4; len < long_chunks; len += len < 16 ? 1 : len < 64 ? 2 : len / 8) {
    const int64_t ids = tile_ids(tokens, n, len * kChunk);
    if (heads * 2 * 512 * (ids + kXcds) >= kMostThreads) continue;
    const double of_long = ceil(long_chunks / len);
    // (others of different lengths end inside a segment, half of one on average)
    const double of_rest = rest_chunks == long_chunks ? of_long : rest_chunks / len + .5;
    const double segs = of_long + (n - 1) * of_rest;
    const double starts = segs - n;  // segments whose end is asked for
    // (Ids of no segment, between those of sequences that end inside one, leave the XCDs
    // uneven loads, the more so the more of them there are: almost as many workgroups as
    // CUs take two rounds then. 9 x 1500 tokens in segments of 8 chunks, 216 workgroups,
    // 235 us for 158 whole; 16 x 2000 in ones of 16, 256 workgroups, 242 for 198.)
    const double uneven = n == 1 || fmod(most, len * kChunk) == 0 ? 1. : n <= 8 ? 1.1 : 1.35;
    const float join = kPassStart + (float)of_long * c.join;
    const float by8 = pass_time(c.ends8, heads * starts * (delta ? 2 : 1), len, cus, uneven);
    const float by16 = pass_time(c.ends16, heads * starts, len, cus, uneven);
    for (int32_t waves = norm ? 8 : 4; waves <= 8; waves += 4) {
      const float (&cost)[2] = norm ? c.normed8 : waves == 4 ? c.rows4 : c.rows8;
      const float t = join + (delta && by16 < by8 ? by16 : by8) +
                      pass_time(cost, heads * (8 / waves) * segs, len, cus, uneven);
      if (t < best) {
        best = t;
        p.waves = waves;
        p.end_waves = delta && by16 < by8 ? 16 : 8;
        p.seg = len * kChunk;
      }
    }
  }
}

Prefill plan_prefill(int64_t tokens, int32_t n, int32_t longest, int32_t hk, int32_t hv,
                     bool delta, bool norm) {
  Prefill p{};
  p.total = kLeastBytes;
  p.chunked = tokens > 0 && n > 0 && (longest == 0 || longest > kScanTokens);
  if (!p.chunked) return p;
  p.ids = tile_ids(tokens, n);
  const int64_t group = hv / hk, head = p.ids * head_image(delta), key = p.ids * kKeyImage;
  const auto within = [](int64_t x, int64_t most) { return x < 1 ? 1 : x < most ? x : most; };
  p.khs = (int32_t)within(kImageBytes / (key + group * head), hk);
  p.vhs = (int32_t)(p.khs > 1 ? group : within((kImageBytes - key) / head, group));
  const int64_t heads = (int64_t)p.khs * p.vhs;
  choose_walk(p, tokens, n, longest, (double)heads, delta, norm);
  if (p.seg) p.segs = tile_ids(tokens, n, p.seg);
  p.key_bytes = p.ids * p.khs * kKeyImage;
  p.head_bytes = p.ids * heads * head_image(delta);
  p.end_bytes = p.segs * heads * kStateHead * 4;
  p.step_bytes = delta ? p.end_bytes : p.segs * heads * 4;
  p.total = p.key_bytes + p.head_bytes + p.end_bytes + p.step_bytes;
  return p;
}

dim3 walk_grid(const LinArgs& a, const ChunkArgs& c) {
  const int64_t pairs = (int64_t)c.khs * c.rows;
  return dim3((unsigned)((pairs + kXcds - 1) / kXcds * kXcds * a.group * c.parts));
}

// The call on some value heads of one key head.
LinArgs some_heads(const LinArgs& all, int32_t kh, int32_t first, int32_t count) {
  LinArgs a = all;
  const int64_t h = (int64_t)kh * all.group + first, gate = all.gates_bf16 ? 2 : 4;
  a.hk = 1;
  a.group = count;  // (hv stays: the strides of states and outputs)
  a.q += kh * (kDim * 2);
  a.k += kh * (kDim * 2);
  a.v += h * (kDim * 2);
  a.g += h * gate;
  if (a.beta) a.beta += h * gate;
  if (a.a_log) a.a_log += h, a.dt_bias += h;
  if (a.z) a.z += h * (kDim * 2);
  a.out += h * (kDim * 2);
  a.state += h * kStateHead;
  return a;
}

template <bool DELTA>
void run_heads(const LinArgs& a, const Prefill& p, uint8_t* ws, hipStream_t s) {
  ChunkArgs c{};
  c.keys = ws;
  c.heads = c.keys + p.key_bytes;
  c.ends = (float*)(c.heads + p.head_bytes);
  c.steps = (float*)((uint8_t*)c.ends + p.end_bytes);
  c.seg = p.seg;
  for (int32_t kh0 = 0; kh0 < a.hk; kh0 += p.khs) {
    c.kh0 = kh0;
    c.khs = a.hk - kh0 < p.khs ? a.hk - kh0 : p.khs;
    const unsigned heads = (unsigned)(c.khs * a.group), n = (unsigned)a.n;
    hipLaunchKernelGGL(linear_prep_kernel<DELTA>, dim3((unsigned)p.ids, (unsigned)c.khs),
                       dim3(DELTA ? kPrepThreads : kPrepThreads / 2), 0, s, a, c);
    if (p.seg) {
      c.rows = (int32_t)p.segs;
      c.parts = DELTA && p.end_waves == 8 ? 2 : 1;  // (with the delta rule M's 128 rows too)
      if (p.end_waves == 16)
        hipLaunchKernelGGL((linear_chunk_kernel<DELTA ? 16 : 8, DELTA, kEnds>), walk_grid(a, c),
                           dim3(DELTA ? 1024 : 512), 0, s, a, c);
      else
        hipLaunchKernelGGL((linear_chunk_kernel<8, DELTA, kEnds>), walk_grid(a, c), dim3(512), 0, s,
                           a, c);
      hipLaunchKernelGGL(linear_join_kernel<DELTA>, dim3(heads * (kDim / 16), n), dim3(256), 0, s,
                         a, c);
    }
    c.parts = 8 / p.waves;
    c.rows = p.seg ? (int32_t)p.segs : a.n;
    const dim3 grid = walk_grid(a, c), block(64 * p.waves);
    if (p.seg && p.waves == 8 && a.z)
      hipLaunchKernelGGL((linear_chunk_kernel<8, DELTA, kRows, true>), grid, block, 0, s, a, c);
    else if (p.seg && p.waves == 8)
      hipLaunchKernelGGL((linear_chunk_kernel<8, DELTA, kRows>), grid, block, 0, s, a, c);
    else if (p.seg)
      hipLaunchKernelGGL((linear_chunk_kernel<4, DELTA, kRows>), grid, block, 0, s, a, c);
    else if (p.waves == 8 && a.z)
      hipLaunchKernelGGL((linear_chunk_kernel<8, DELTA, kWhole, true>), grid, block, 0, s, a, c);
    else if (p.waves == 8)
      hipLaunchKernelGGL((linear_chunk_kernel<8, DELTA, kWhole>), grid, block, 0, s, a, c);
    else
      hipLaunchKernelGGL((linear_chunk_kernel<4, DELTA, kWhole>), grid, block, 0, s, a, c);
  }
}

template <bool DELTA>
void run_chunks(const LinArgs& a, const Prefill& p, uint8_t* ws, hipStream_t s) {
  if (p.vhs == a.group) return run_heads<DELTA>(a, p, ws, s);
  for (int32_t kh = 0; kh < a.hk; ++kh)
    for (int32_t o = 0; o < a.group; o += p.vhs)
      run_heads<DELTA>(some_heads(a, kh, o, a.group - o < p.vhs ? a.group - o : p.vhs), p, ws, s);
}

}  // namespace
}  // namespace mkv

extern "C" int64_t mkv_linear_attn_prefill_workspace_bytes(int64_t num_tokens, int32_t batch,
                                                           int32_t max_seqlen, int32_t num_k_heads,
                                                           int32_t num_v_heads, int32_t delta) {
  if (num_tokens < 0 || num_tokens >= (1ll << 31) || batch < 0 || max_seqlen < 0 ||
      num_k_heads <= 0 || num_v_heads <= 0 || num_v_heads % num_k_heads != 0)
    return -1;
  // (with and without the output norm: its walk may have other segments)
  int64_t most = 0;
  for (const bool norm : {false, true}) {
    const int64_t bytes =
        plan_prefill(num_tokens, batch, max_seqlen, num_k_heads, num_v_heads, delta != 0, norm).total;
    most = bytes > most ? bytes : most;
  }
  return most;
}

extern "C" int mkv_linear_attn_prefill(
    void* state, int64_t pool_slots, int32_t num_k_heads, int32_t num_v_heads, int32_t head_dim,
    const int32_t* slots, const int32_t* cu_seqlens, int32_t batch, int64_t num_tokens,
    int32_t max_seqlen, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
    const void* v, int64_t v_stride, const void* g, int64_t g_stride, const void* beta,
    int64_t beta_stride, int32_t gates_bf16, const float* a_log, const float* dt_bias,
    int32_t qk_norm, float scale, const void* z, int64_t z_stride, const void* norm_weight,
    int32_t weight_bf16, float norm_eps, void* out, void* workspace, int64_t workspace_bytes,
    int32_t* err, void* stream) {
  clear_error();
  const char* fn = "mkv_linear_attn_prefill";
  LinArgs a{};
  const int rc = linear_args(fn, state, pool_slots, num_k_heads, num_v_heads, head_dim, slots,
                             batch, num_tokens, q, q_stride, k, k_stride, v, v_stride, g, g_stride,
                             beta, beta_stride, gates_bf16, a_log, dt_bias, qk_norm, scale, z,
                             z_stride, norm_weight, weight_bf16, norm_eps, out, err, a);
  if (rc != MKV_OK) return rc;
  MKV_REQUIRE(num_tokens < (1ll << 31) && max_seqlen >= 0, MKV_E_INVALID, "%s: bad sizes", fn);
  MKV_REQUIRE(batch <= kMaxSequences, MKV_E_UNSUPPORTED, "%s: more than %d sequences", fn,
              kMaxSequences);
  MKV_REQUIRE(num_tokens <= kNormMaxRows / num_v_heads, MKV_E_UNSUPPORTED, "%s: too many rows", fn);
  MKV_REQUIRE(v_stride <= kMostStride, MKV_E_UNSUPPORTED, "%s: rows of v more than 16 MiB apart", fn);
  if (batch == 0 || num_tokens == 0) return MKV_OK;
  const Prefill p =
      plan_prefill(num_tokens, batch, max_seqlen, num_k_heads, num_v_heads, beta != nullptr,
                   z != nullptr);
  // (the walk's grids stay within theirs: whole sequences have at most 2^31 threads)
  MKV_REQUIRE((double)p.ids * kPrepThreads < kMostThreads, MKV_E_UNSUPPORTED, "%s: too many rows",
              fn);
  MKV_REQUIRE(cu_seqlens && workspace && aligned4(cu_seqlens), MKV_E_INVALID, "%s: null pointer",
              fn);
  MKV_REQUIRE(aligned16(workspace) && workspace_bytes >= p.total, MKV_E_INVALID,
              "%s: the workspace must be 16-byte aligned and hold %lld bytes", fn,
              (long long)p.total);
  a.cu = cu_seqlens;
  const hipStream_t s = as_stream(stream);
  const dim3 scan((unsigned)num_v_heads * (a.z ? 1 : 2), (unsigned)batch);
  if (!p.chunked && a.z)
    hipLaunchKernelGGL(linear_scan_kernel<true>, scan, dim3(256), 0, s, a);
  else if (!p.chunked)
    hipLaunchKernelGGL(linear_scan_kernel<false>, scan, dim3(256), 0, s, a);
  else if (a.beta)
    run_chunks<true>(a, p, (uint8_t*)workspace, s);
  else
    run_chunks<false>(a, p, (uint8_t*)workspace, s);
  return check_launch(fn);
}

extern "C" int mkv_gated_rms_norm(const void* x, int64_t x_stride, const void* z, int64_t z_stride,
                                  int64_t tokens, int32_t heads, int32_t dim, const void* weight,
                                  int32_t weight_bf16, float eps, void* out, void* stream) {
  clear_error();
  const char* fn = "mkv_gated_rms_norm";
  MKV_REQUIRE(tokens >= 0 && heads > 0 && dim > 0, MKV_E_INVALID, "%s: bad sizes", fn);
  MKV_REQUIRE(dim % 8 == 0 && dim <= kNormMaxDim, MKV_E_UNSUPPORTED,
              "%s: rows of %d values unsupported (a multiple of 8, at most %d)", fn, dim,
              kNormMaxDim);
  if (tokens == 0) return MKV_OK;
  MKV_REQUIRE(x && z && weight && out, MKV_E_INVALID, "%s: null pointer", fn);
  const int64_t row = (int64_t)heads * dim * 2;
  MKV_REQUIRE(x_stride >= row && z_stride >= row, MKV_E_INVALID,
              "%s: a stride is shorter than its row", fn);
  MKV_REQUIRE(aligned16(x) && aligned16(z) && aligned16(out) && x_stride % 16 == 0 &&
                  z_stride % 16 == 0 && (uintptr_t)weight % (weight_bf16 ? 2 : 4) == 0,
              MKV_E_ALIGN, "%s: rows must be 16-byte aligned, the weight to its type", fn);
  MKV_REQUIRE(tokens <= kNormMaxRows / heads, MKV_E_UNSUPPORTED, "%s: too many rows", fn);
  NormArgs a{(const uint8_t*)x, (const uint8_t*)z, (const uint8_t*)weight, x_stride, z_stride,
             heads, dim, weight_bf16, eps, (uint8_t*)out, tokens * heads};
  run_norm(a, as_stream(stream));
  return check_launch(fn);
}
