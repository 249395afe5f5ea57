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
__device__ __forceinline__ void load4(const uint8_t* p, float (&x)[4]) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 w = *(const u32x2*)p;
  x[0] = bits_f32(w.x << 16);
  x[1] = bits_f32(w.x & 0xffff0000u);
  x[2] = bits_f32(w.y << 16);
  x[3] = bits_f32(w.y & 0xffff0000u);
}

// sum over the 8 lanes that share a row of the state
__device__ __forceinline__ float sum8(float x) {
  x += __shfl_xor(x, 1);
  x += __shfl_xor(x, 2);
  x += __shfl_xor(x, 4);
  return x;
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
    m = sum8(m);
    rk = rq = 1.f;
    if (a.qk_norm) {
      rk = 1.f / sqrtf(sum8(kk) + kL2Eps);
      rq = 1.f / sqrtf(sum8(qq) + kL2Eps);
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
      x = sum8(x);
      y = sum8(y);
      const float u = a.beta ? beta * (v[i] - e * rk * x) : v[i];
      o[i] = a.scale * (e * rq * y + u * kq);
      const float w = u * rk;
#pragma unroll
      for (int j = 0; j < 16; ++j) s[i][j] = fmaf(w, kx[j], e * s[i][j]);
    }
  }
};

__device__ __forceinline__ float silu(float x) { return x / (1.f + expf(-x)); }

__device__ __forceinline__ float weight_at(const uint8_t* w, int32_t bf16, int64_t i) {
  return bf16 ? bf16_at(w + 2 * i) : *(const float*)(w + 4 * i);
}

// One workgroup per (value head, request): the head's 64 KiB state is read
// once, updated in registers and written back. Bound by HBM: 128 KiB per
// (request, head) against 0.8 KiB of everything else.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void linear_decode_kernel(LinArgs a) {
  constexpr int kGroups = THREADS / 8, kRows = kDim / kGroups;
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
      const u32x4 x = ld16((const uint8_t*)(st + (r0 + kGroups * i) * kDim + 32 * c + 4 * l));
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
      st16((uint8_t*)(st + (r0 + kGroups * i) * kDim + 32 * c + 4 * l), x);
    }
  if (a.z) {  // uniform: o / sqrt(mean(o^2) + eps) w silu(z)
    __shared__ float part[THREADS / 64];
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) q = fmaf(o[i], o[i], q);
    q += __shfl_xor(q, 8);
    q += __shfl_xor(q, 16);
    q += __shfl_xor(q, 32);
    if ((tid & 63) == 0) part[tid >> 6] = q;
    __syncthreads();
    q = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) q += part[i];
    const float r = 1.f / sqrtf(q * (1.f / kDim) + a.eps);
    const uint8_t* zp = a.z + b * a.z_stride + h * (kDim * 2);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int d = r0 + kGroups * i;
      o[i] = o[i] * r * weight_at(a.w, a.w_bf16, d) * silu(bf16_at(zp + 2 * d));
    }
  }
  if (l == 0) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      *(uint16_t*)(out + 2 * (r0 + kGroups * i)) = f32_to_bf16_rne(o[i]);
  }
}

// ---------------------------------------------------------------------------
// Prompts
// ---------------------------------------------------------------------------

// One workgroup per 64 value dims of a (head, sequence), token after token.
__global__ __launch_bounds__(256) void linear_scan_kernel(LinArgs a, int32_t* ok_word) {
  constexpr int kRows = 2;
  const int tid = threadIdx.x, l = tid & 7, r0 = tid >> 3;
  const int32_t h = blockIdx.x >> 1, kh = h / a.group, d0 = (blockIdx.x & 1) * 64;
  const int32_t b = blockIdx.y;
  const bool first = blockIdx.x == 0 && tid == 0;
  const bool ok = offsets_ok(a.cu, a.n, a.tokens);
  if (first && b == 0) *ok_word = ok;
  if (!ok) {
    if (first && b == 0) raise_err(a.err, MKV_DEVERR_TABLE);
    return;
  }
  const int64_t t0 = a.cu[b], t1 = a.cu[b + 1];
  const int32_t slot = a.slots[b];
  if (slot < 0 || slot >= a.pool_slots) {  // uniform
    if (first) raise_err(a.err, MKV_DEVERR_STATE_SLOT);
    for (int64_t t = t0 + (tid >> 5); t < t1; t += 8)
      *(uint32_t*)(a.out + (t * a.hv + h) * (kDim * 2) + d0 * 2 + 4 * (tid & 31)) = 0u;
    return;
  }
  if (t0 == t1) return;
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
  for (int64_t t = t0; t < t1; ++t) {
    float g, beta, v[kRows], o[kRows];
    m.keys(a, t, kh, l);
    load_gates(a, t, h, g, beta);
    const uint8_t* vp = a.v + t * a.v_stride + (h * kDim + d0) * 2;
#pragma unroll
    for (int i = 0; i < kRows; ++i) v[i] = bf16_at(vp + 2 * (r0 + 32 * i));
    m.norms(a);
    m.step(a, g, beta, v, o);
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
// y = x / sqrt(mean(x^2) + eps) w silu(z), a row of `dim` values at a time
// ---------------------------------------------------------------------------
struct NormArgs {
  const uint8_t *x, *z, *w;
  int64_t x_stride, z_stride;  // bytes between tokens; a token's heads follow each other
  int32_t heads, dim, w_bf16;
  float eps;
  uint8_t* out;  // [tokens, heads, dim]
  int64_t rows;  // tokens * heads
  const int32_t* cu;  // with n: only the tokens of cu[0] .. cu[n] - 1, if *ok
  int32_t n;
  const int32_t* ok;
};

// LANES lanes per row, 8 values (16 bytes) per lane and step.
template <int LANES, int STEPS>
__global__ __launch_bounds__(kThreads) void gated_norm_kernel(NormArgs a) {
  constexpr int kRowsPerWg = kThreads / LANES;
  const int lane = threadIdx.x % LANES;
  const int64_t row = (int64_t)blockIdx.x * kRowsPerWg + threadIdx.x / LANES;
  const bool there = row < a.rows;
  const int64_t at = there ? row : 0;
  const int64_t token = a.heads == 1 ? at : at / a.heads;
  const int64_t head = at - token * a.heads;
  if (a.cu) {  // rows outside the sequences stay as they are
    if (!*a.ok || !there || token < a.cu[0] || token >= a.cu[a.n]) return;
  } else if (!there) {
    return;
  }
  const uint8_t* xp = a.x + token * a.x_stride + head * a.dim * 2;
  const uint8_t* zp = a.z + token * a.z_stride + head * a.dim * 2;
  u32x4 xv[STEPS], zv[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int d = (s * LANES + lane) * 8;
    xv[s] = zv[s] = u32x4{0u, 0u, 0u, 0u};
    if (d < a.dim) {
      xv[s] = ld16(xp + 2 * d);
      zv[s] = ld16(zp + 2 * d);
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
#pragma unroll
  for (int o = 1; o < LANES; o *= 2) q += __shfl_xor(q, o);
  const float r = 1.f / sqrtf(q / (float)a.dim + a.eps);
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int d = (s * LANES + lane) * 8;
    if (d >= a.dim) continue;
    u32x4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x0 = bits_f32(xv[s][j] << 16), x1 = bits_f32(xv[s][j] & 0xffff0000u);
      const float z0 = bits_f32(zv[s][j] << 16), z1 = bits_f32(zv[s][j] & 0xffff0000u);
      const float y0 = x0 * r * weight_at(a.w, a.w_bf16, d + 2 * j) * silu(z0);
      const float y1 = x1 * r * weight_at(a.w, a.w_bf16, d + 2 * j + 1) * silu(z1);
      y[j] = (uint32_t)f32_to_bf16_rne(y0) | ((uint32_t)f32_to_bf16_rne(y1) << 16);
    }
    st16(a.out + (row * a.dim + d) * 2, y);
  }
}

template <int LANES, int STEPS>
void launch_norm(const NormArgs& a, hipStream_t stream) {
  constexpr int kRowsPerWg = kThreads / LANES;
  hipLaunchKernelGGL((gated_norm_kernel<LANES, STEPS>),
                     dim3((unsigned)((a.rows + kRowsPerWg - 1) / kRowsPerWg)), dim3(kThreads), 0,
                     stream, a);
}

constexpr int kNormMaxDim = 4096;

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
  hipLaunchKernelGGL(linear_decode_kernel<256>, grid, dim3(256), 0, as_stream(stream), a);
  return check_launch(fn);
}

namespace mkv {
namespace {
constexpr int64_t kHeadBytes = 16;  // the workspace's first bytes: the offsets' verdict
}
}  // namespace mkv

extern "C" int64_t mkv_linear_attn_prefill_workspace_bytes(int64_t num_tokens, int32_t batch,
                                                           int32_t max_seqlen, int32_t num_k_heads,
                                                           int32_t num_v_heads, int32_t delta) {
  if (num_tokens < 0 || batch < 0 || max_seqlen < 0 || num_k_heads <= 0 || num_v_heads <= 0)
    return -1;
  return kHeadBytes;
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
  if (batch == 0 || num_tokens == 0) return MKV_OK;
  const int64_t need = mkv_linear_attn_prefill_workspace_bytes(
      num_tokens, batch, max_seqlen, num_k_heads, num_v_heads, beta != nullptr);
  MKV_REQUIRE(cu_seqlens && workspace && aligned4(cu_seqlens), MKV_E_INVALID, "%s: null pointer",
              fn);
  MKV_REQUIRE(aligned16(workspace) && workspace_bytes >= need, MKV_E_INVALID,
              "%s: the workspace must be 16-byte aligned and hold %lld bytes", fn,
              (long long)need);
  a.cu = cu_seqlens;
  const hipStream_t s = as_stream(stream);
  int32_t* ok = (int32_t*)workspace;
  hipLaunchKernelGGL(linear_scan_kernel, dim3((unsigned)num_v_heads * 2, (unsigned)batch),
                     dim3(256), 0, s, a, ok);
  const int launched = check_launch(fn);
  if (launched != MKV_OK || !a.z) return launched;
  NormArgs m{a.out, a.z, a.w, (int64_t)a.hv * kDim * 2, a.z_stride, a.hv, kDim, a.w_bf16, a.eps,
             a.out, num_tokens * a.hv, a.cu, a.n, ok};
  run_norm(m, s);
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
  MKV_REQUIRE(tokens <= (1ll << 32) / heads, MKV_E_UNSUPPORTED, "%s: too many rows", fn);
  NormArgs a{(const uint8_t*)x, (const uint8_t*)z, (const uint8_t*)weight, x_stride, z_stride,
             heads, dim, weight_bf16, eps, (uint8_t*)out, tokens * heads, nullptr, 0, nullptr};
  run_norm(a, as_stream(stream));
  return check_launch(fn);
}
