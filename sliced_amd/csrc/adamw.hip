// AdamW over many parameter tensors at once, with its two moments in f32 or in 8 bits.
//
//   m = b1*m + (1-b1)*g            v = b2*v + (1-b2)*g*g
//   p = p*(1 - lr*wd) - lr/(1-b1^t) * m / (sqrt(v)/sqrt(1-b2^t) + eps)
//
// Every element is read and written once and nothing is reduced but the blocks' largest magnitudes, so
// HBM is the bound: 28 bytes an element with f32 moments (p, m, v in and out, g in), 16 with 8-bit ones.  Measured: 40 M
// elements in 150 tensors 190 us (5.9 TB/s, three launches), 134 M with 8-bit moments 345 us (6.2 TB/s), 5.8 M 19.5 us (4.8),
// the six tensors of a net of 4353 parameters 3.1 us in the kernel.
//
// A launch takes up to 64 tensors: their pointers and the number of each one's first workgroup travel in
// the kernel arguments, and a workgroup finds its tensor with one load and one ballot - lane i compares
// its number with tensor i's first workgroup - where a search would chain six loads.  Tensors of any
// mix of lengths so fill the chip as one flat list of tiles.
//
// 8-bit moments.  m is kept as OCP E4M3 and v as OCP E5M2, in blocks of 256 elements with one scale each, a
// power of two: scaling is then exact both ways and the only rounding is to the 8-bit format.  (A float
// format wants the scale for its range, not for its precision: a power of two loses nothing.)  m is rounded
// to nearest.  v is rounded stochastically: at b2 = 0.999 its decay of 0.1 % a step is far below half the
// spacing of any 8-bit format, so rounded to nearest it would never decay.  (m's decay of 10 % is more than half the spacing
// down to four units of the smallest, 2^-14 of the block's largest m; what is below that stays, while that one does.)  The random bits come from the
// counter-based generator of slhip_rand_uniform, keyed by seed, step, tensor and element, so a step is
// reproducible.  A v that is not zero is kept at the format's smallest value or above, never at zero: with
// an m that is still there, zero would make the next update m / eps.  The update itself uses the moments
// before they are rounded.
#include "common.hpp"

#include <algorithm>
#include <cmath>
#include <new>

namespace slhip {

constexpr int ADAMW_TENSORS = 64;   // of one launch: a lane each in the search for a workgroup's tensor
constexpr int ADAMW_BLOCK = 256;    // elements of a scale: a wave's 64 lanes hold four each
constexpr int ADAMW_ROWS = 2;       // blocks of 256 elements a wave takes (1, 2, 3, 4 of them: 134 M elements with 8-bit
                                    // moments 370, 348, 350, 355 us, 5.8 M 19.7, 19.7, 20.2, 21.9, 40 M with f32 ones 188, 189, 196, 206)
constexpr size_t ADAMW_TILE = (size_t)4 * ADAMW_ROWS * ADAMW_BLOCK;  // elements of a workgroup of four waves
constexpr size_t ADAMW_LONGEST = MAX_GRID / ADAMW_TENSORS * ADAMW_TILE;  // elements of a tensor: 64 of them fit a launch

// What depends on the number of the step: passed by value, or left in the workspace by adamw_advance_kernel.
struct AdamwStep {
  float size;     // lr / (1 - b1^t)
  float root;     // 1 / sqrt(1 - b2^t)
  uint64_t bits;  // of the random words: splitmix64(seed + t)
};

struct AdamwRates {
  float b1, r1, b2, r2, keep, eps;  // r = 1 - b, keep = 1 - lr*wd
};

struct AdamwArgs {
  float* p[ADAMW_TENSORS];
  const float* g[ADAMW_TENSORS];
  float* m[ADAMW_TENSORS];
  float* v[ADAMW_TENSORS];
  size_t n[ADAMW_TENSORS];
  unsigned first[ADAMW_TENSORS];  // number of the tensor's first workgroup; ~0u behind the last tensor
  AdamwRates r;
  AdamwStep step;
  const AdamwStep* step_dev;  // or null
};

struct Adamw8Args {
  float* p[ADAMW_TENSORS];
  const float* g[ADAMW_TENSORS];
  uint8_t* m[ADAMW_TENSORS];
  uint8_t* v[ADAMW_TENSORS];
  float* scales[ADAMW_TENSORS];
  size_t n[ADAMW_TENSORS];
  unsigned first[ADAMW_TENSORS];
  unsigned ordinal;  // of tensor 0 in the caller's list
  AdamwRates r;
  AdamwStep step;
  const AdamwStep* step_dev;
};
static_assert(sizeof(AdamwArgs) <= 4096 && sizeof(Adamw8Args) <= 4096, "kernel arguments");

__host__ __device__ __forceinline__ uint64_t adamw_mix(uint64_t s) {  // splitmix64
  uint64_t z = s + 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}

__host__ __device__ __forceinline__ AdamwStep adamw_step_of(uint64_t t, double lr, double b1, double b2, uint64_t seed) {
  // in 64 bits: b^t of a late step and 1 - b^t of an early one both lose too much in 32
  AdamwStep s;
  s.size = (float)(lr / (1.0 - pow(b1, (double)t)));
  s.root = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
  s.bits = adamw_mix(seed + t);
  return s;
}

// Advances a step counter that lives on the device, for steps that a recording replays.
__global__ __launch_bounds__(64) void adamw_advance_kernel(uint64_t* counter, float lr, float b1, float b2, uint64_t seed,
                                                           AdamwStep* out) {
  if (threadIdx.x != 0) return;
  const uint64_t t = *counter + 1;
  *counter = t;
  *out = adamw_step_of(t, lr, b1, b2, seed);
}

// The tensor of this workgroup: how many tensors start at or before it, less one.
__device__ __forceinline__ int adamw_tensor(const unsigned* first) {
  const unsigned mine = first[threadIdx.x & 63];
  return __popcll(__ballot(blockIdx.x >= mine)) - 1;
}

__device__ __forceinline__ void adamw_element(float& p, float g, float& m, float& v, const AdamwRates& r, float size, float root) {
  m = m * r.b1 + g * r.r1;
  v = v * r.b2 + (g * r.r2) * g;
  p = p * r.keep - size * (m / (sqrtf(v) * root + r.eps));
}

__global__ __launch_bounds__(256) void adamw_kernel(AdamwArgs a) {
  const int t = adamw_tensor(a.first);
  float* const p = a.p[t];
  const float* const g = a.g[t];
  float* const m = a.m[t];
  float* const v = a.v[t];
  const size_t n = a.n[t];
  const size_t i0 = (size_t)(blockIdx.x - a.first[t]) * ADAMW_TILE + 4 * threadIdx.x;
  AdamwStep s = a.step;
  if (a.step_dev) s = *a.step_dev;
  float4 pv[ADAMW_ROWS], gv[ADAMW_ROWS], mv[ADAMW_ROWS], vv[ADAMW_ROWS];
#pragma unroll
  for (int u = 0; u < ADAMW_ROWS; ++u) {
    const size_t i = i0 + (size_t)u * 1024;
    if (i + 3 < n) {
      pv[u] = ld4s(p + i); gv[u] = ld4s(g + i); mv[u] = ld4s(m + i); vv[u] = ld4s(v + i);
    }
  }
#pragma unroll
  for (int u = 0; u < ADAMW_ROWS; ++u) {
    const size_t i = i0 + (size_t)u * 1024;
    if (i + 3 < n) {
      adamw_element(pv[u].x, gv[u].x, mv[u].x, vv[u].x, a.r, s.size, s.root);
      adamw_element(pv[u].y, gv[u].y, mv[u].y, vv[u].y, a.r, s.size, s.root);
      adamw_element(pv[u].z, gv[u].z, mv[u].z, vv[u].z, a.r, s.size, s.root);
      adamw_element(pv[u].w, gv[u].w, mv[u].w, vv[u].w, a.r, s.size, s.root);
      st4s(p + i, pv[u]); st4s(m + i, mv[u]); st4s(v + i, vv[u]);
    } else {
      for (size_t j = i; j < n && j < i + 4; ++j) {
        float pe = p[j], me = m[j], ve = v[j];
        adamw_element(pe, g[j], me, ve, a.r, s.size, s.root);
        p[j] = pe; m[j] = me; v[j] = ve;
      }
    }
  }
}

// ---------------------------------------------------------------- 8-bit moments
// Largest value over the wave of two 16-bit halves at once, in lane 63: row shifts by 1, 2, 4, 8, then the
// broadcasts of a row's last lane to the next row and of lane 31 to the upper half.
typedef unsigned short adamw_u16x2 __attribute__((ext_vector_type(2)));
template <int CTRL>
__device__ __forceinline__ unsigned adamw_max_step(unsigned x) {
  const unsigned y = (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
  adamw_u16x2 a, b;
  __builtin_memcpy(&a, &x, 4);
  __builtin_memcpy(&b, &y, 4);
  a = __builtin_elementwise_max(a, b);
  __builtin_memcpy(&x, &a, 4);
  return x;
}
__device__ __forceinline__ unsigned adamw_wave_max(unsigned x) {
  x = adamw_max_step<0x111>(x);  // row_shr:1
  x = adamw_max_step<0x112>(x);
  x = adamw_max_step<0x114>(x);
  x = adamw_max_step<0x118>(x);
  x = adamw_max_step<0x142>(x);  // row_bcast:15
  x = adamw_max_step<0x143>(x);  // row_bcast:31
  return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}

// Exponent field of a finite value, 0 for infinity and NaN: those are stored as what they are and have no say in the scale.
__device__ __forceinline__ unsigned adamw_exponent(float x) {
  const unsigned e = (__float_as_uint(x) >> 23) & 0xffu;
  return e == 0xffu ? 0u : e;
}

// v's value in units of its scale, stochastically rounded to E5M2: r16 / 2^16 of the format's spacing is added before the
// rest is cut off.  That spacing is a quarter of the leading bit down to the smallest normal value, 2^-14, and 2^-16 below it;
// with 2^-14 added a value from below lies in the binade whose quarter is 2^-16, so that one cut does for both.  What is left
// is what the format holds: the conversion rounds nothing.  (Two bits behind the leading one everywhere, the rest left to the
// conversion, would round twice below 2^-14, the second time to nearest: 2 and 4 units of 2^-16 then never decay.)  y = v / scale is zero
// where v is some 2^164 below the block's largest: whether there is a v is asked of v itself.
__device__ __forceinline__ float adamw_round_v(float v, float y, unsigned r16) {
  const float o = y < 6.103515625e-05f ? 6.103515625e-05f : 0.0f;  // 2^-14
  const float cut = __uint_as_float((__float_as_uint(y + o) + (r16 << 5)) & ~0x1fffffu) - o;
  return v > 0.0f && y < __builtin_huge_valf() ? fmaxf(cut, 1.52587890625e-05f) : y;  // 2^-16, E5M2's smallest
}

__global__ __launch_bounds__(256) void adamw8_kernel(Adamw8Args a) {
  const int t = adamw_tensor(a.first);
  float* const p = a.p[t];
  const float* const g = a.g[t];
  uint8_t* const m8 = a.m[t];
  uint8_t* const v8 = a.v[t];
  float* const scales = a.scales[t];
  const size_t n = a.n[t];
  const int lane = threadIdx.x & 63;
  AdamwStep s = a.step;
  if (a.step_dev) s = *a.step_dev;
  const uint64_t key = adamw_mix(s.bits + (uint64_t)(a.ordinal + (unsigned)t));
  const size_t block0 = (size_t)(blockIdx.x - a.first[t]) * (4 * ADAMW_ROWS) + (threadIdx.x >> 6);
  float pv[ADAMW_ROWS][4], gv[ADAMW_ROWS][4];
  unsigned mq[ADAMW_ROWS], vq[ADAMW_ROWS];
  float sm[ADAMW_ROWS], sv[ADAMW_ROWS];
  // what lies behind the end of the tensor counts as zeros, which no scale notices
#pragma unroll
  for (int u = 0; u < ADAMW_ROWS; ++u) {
    const size_t block = block0 + 4 * u, i = block * ADAMW_BLOCK + 4 * lane;
    mq[u] = vq[u] = 0;
    sm[u] = sv[u] = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) pv[u][k] = gv[u][k] = 0.0f;
    if (i + 3 < n) {
      const float4 x = ld4s(p + i), y = ld4s(g + i);
      pv[u][0] = x.x; pv[u][1] = x.y; pv[u][2] = x.z; pv[u][3] = x.w;
      gv[u][0] = y.x; gv[u][1] = y.y; gv[u][2] = y.z; gv[u][3] = y.w;
      mq[u] = __builtin_nontemporal_load(reinterpret_cast<const unsigned*>(m8 + i));
      vq[u] = __builtin_nontemporal_load(reinterpret_cast<const unsigned*>(v8 + i));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) {
          pv[u][k] = p[i + k];
          gv[u][k] = g[i + k];
          mq[u] |= (unsigned)m8[i + k] << (8 * k);
          vq[u] |= (unsigned)v8[i + k] << (8 * k);
        }
    }
    if (block * ADAMW_BLOCK < n) {
      sm[u] = scales[2 * block];
      sv[u] = scales[2 * block + 1];
    }
  }
#pragma unroll
  for (int u = 0; u < ADAMW_ROWS; ++u) {
    const size_t block = block0 + 4 * u, i = block * ADAMW_BLOCK + 4 * lane;
    float m[4], v[4];
    m[0] = __builtin_amdgcn_cvt_f32_fp8((int)mq[u], 0) * sm[u];
    m[1] = __builtin_amdgcn_cvt_f32_fp8((int)mq[u], 1) * sm[u];
    m[2] = __builtin_amdgcn_cvt_f32_fp8((int)mq[u], 2) * sm[u];
    m[3] = __builtin_amdgcn_cvt_f32_fp8((int)mq[u], 3) * sm[u];
    v[0] = __builtin_amdgcn_cvt_f32_bf8((int)vq[u], 0) * sv[u];
    v[1] = __builtin_amdgcn_cvt_f32_bf8((int)vq[u], 1) * sv[u];
    v[2] = __builtin_amdgcn_cvt_f32_bf8((int)vq[u], 2) * sv[u];
    v[3] = __builtin_amdgcn_cvt_f32_bf8((int)vq[u], 3) * sv[u];
    unsigned em = 0, ev = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      adamw_element(pv[u][k], gv[u][k], m[k], v[k], a.r, s.size, s.root);
      const unsigned x = adamw_exponent(m[k]), y = adamw_exponent(v[k]);
      em = em > x ? em : x;
      ev = ev > y ? ev : y;
    }
    // scales that take the block's largest m into [2^7, 2^8) and its largest v into [2^14, 2^15): one binade below the
    // formats' last, so that nothing rounds up past their end.  Kept normal, their reciprocals too.
    const unsigned top = adamw_wave_max((em << 16) | ev);
    const unsigned fm = (top >> 16) > 8u ? (top >> 16) - 7u : 1u, fv = (top & 0xffffu) > 15u ? (top & 0xffffu) - 14u : 1u;
    const float im = __uint_as_float((254u - fm) << 23), iv = __uint_as_float((254u - fv) << 23);
    const uint64_t word = adamw_mix(key + i / 4);
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = adamw_round_v(v[k], v[k] * iv, (unsigned)(word >> (16 * k)) & 0xffffu);
    int mc = __builtin_amdgcn_cvt_pk_fp8_f32(m[0] * im, m[1] * im, 0, false);
    mc = __builtin_amdgcn_cvt_pk_fp8_f32(m[2] * im, m[3] * im, mc, true);
    int vc = __builtin_amdgcn_cvt_pk_bf8_f32(y[0], y[1], 0, false);
    vc = __builtin_amdgcn_cvt_pk_bf8_f32(y[2], y[3], vc, true);
    if (i + 3 < n) {
      st4s(p + i, make_float4(pv[u][0], pv[u][1], pv[u][2], pv[u][3]));
      __builtin_nontemporal_store((unsigned)mc, reinterpret_cast<unsigned*>(m8 + i));
      __builtin_nontemporal_store((unsigned)vc, reinterpret_cast<unsigned*>(v8 + i));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) {
          p[i + k] = pv[u][k];
          m8[i + k] = (uint8_t)((unsigned)mc >> (8 * k));
          v8[i + k] = (uint8_t)((unsigned)vc >> (8 * k));
        }
    }
    if (lane == 0 && block * ADAMW_BLOCK < n) {
      scales[2 * block] = __uint_as_float(fm << 23);
      scales[2 * block + 1] = __uint_as_float(fv << 23);
    }
  }
}

// The arrays of a call, in the order of their addresses: 2^47 of those and 2^17 arrays make one 64-bit key.  Sorting those takes 2 us for 64
// tensors and 14 for 400 whose lists are in address order, 15 and 110 where they are in any order.
constexpr size_t ADAMW_MOST = 16384;  // tensors of a call
static_assert(5 * ADAMW_MOST + 1 <= (size_t(1) << 17), "arrays of a call");

// Whether an array that the call writes shares memory with any other.  `arrays` kinds of `count` pointers each; bytes(kind, i)
// is an array's length, `read_only` the kind that is not written.  The counter of steps, if there is one, comes behind them.
template <class F>
static int32_t adamw_overlap(const char* who, const void* const* const* arrays, int kinds, int read_only, size_t count, const uint64_t* counter,
                             F&& bytes) {
  uint64_t few[5 * ADAMW_TENSORS + 1];
  uint64_t* keys = few;
  const size_t all = count * (size_t)kinds, n = all + (counter ? 1 : 0);
  if (count > ADAMW_TENSORS && !(keys = new (std::nothrow) uint64_t[n])) {
    set_error("%s: out of host memory", who);
    return SLHIP_EINVAL;
  }
  size_t k = 0;
  uint64_t high = 0;
  auto take = [&](const void* p) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    high |= at >> 47;
    keys[k] = at << 17 | k;
    ++k;
  };
  for (int kind = 0; kind < kinds; ++kind)
    for (size_t i = 0; i < count; ++i) take(arrays[kind][i]);
  if (counter) take(counter);
  std::sort(keys, keys + n);
  uint64_t any = 0, written = 0;  // where the arrays so far end, and those of them that are written
  bool shared = false;
  for (size_t i = 0; i < n; ++i) {
    const uint64_t at = keys[i] >> 17, which = keys[i] & ((1u << 17) - 1);
    const int kind = (int)(which / count);
    const uint64_t end = at + (which == all ? sizeof(uint64_t) : bytes(kind, (size_t)(which % count)));
    const bool writes = kind != read_only;
    shared = shared || at < (writes ? any : written);
    if (any < end) any = end;
    if (writes && written < end) written = end;
  }
  if (keys != few) delete[] keys;
  if (high) {
    set_error("%s: not a device address", who);
    return SLHIP_EINVAL;
  }
  if (!shared) return SLHIP_OK;
  set_error("%s: two tensors overlap", who);
  return SLHIP_EALIAS;
}

// Checks what both forms share and fills in the rates; the step of the call comes from the host or, where
// a counter on the device is given, from the workspace (one launch that advances the counter).
static int32_t adamw_begin(slhip_ctx* ctx, const char* who, float lr, float beta1, float beta2, float eps, float weight_decay,
                           uint64_t step, uint64_t* step_dev, uint64_t seed, AdamwRates* r, AdamwStep* s, const AdamwStep** s_dev) {
  if (!(std::isfinite(lr) && std::isfinite(weight_decay) && beta1 >= 0.0f && beta1 < 1.0f && beta2 >= 0.0f && beta2 < 1.0f &&
        eps >= 0.0f && std::isfinite(eps))) {
    set_error("%s: lr, weight_decay and eps must be finite, eps >= 0, beta1 and beta2 in [0, 1)", who);
    return SLHIP_EINVAL;
  }
  if ((step == 0) == (step_dev == nullptr)) {
    set_error("%s: either step (from 1) or step_dev, not both", who);
    return SLHIP_EINVAL;
  }
  if (step_dev && ((uintptr_t)step_dev & 7)) {
    set_error("%s: step_dev must be 8-byte aligned", who);
    return SLHIP_EINVAL;
  }
  *r = AdamwRates{beta1, 1.0f - beta1, beta2, 1.0f - beta2, (float)(1.0 - (double)lr * (double)weight_decay), eps};
  *s = AdamwStep{0.0f, 0.0f, 0};
  *s_dev = nullptr;
  if (!step_dev) {
    *s = adamw_step_of(step, lr, beta1, beta2, seed);
    return SLHIP_OK;
  }
  if (ctx->workspace_bytes < sizeof(AdamwStep)) {
    set_error("%s: workspace too small", who);
    return SLHIP_EWORKSPACE;
  }
  AdamwStep* const at = (AdamwStep*)ctx->workspace;
  hipLaunchKernelGGL(adamw_advance_kernel, dim3(1), dim3(64), 0, ctx->stream, step_dev, lr, beta1, beta2, seed, at);
  *s_dev = at;
  return post_launch();
}

// Numbers the workgroups of tensors first .. first + m and returns how many there are.
template <class Args>
static size_t adamw_number(Args& a, const size_t* lens, size_t m) {
  size_t blocks = 0;
  for (size_t i = 0; i < (size_t)ADAMW_TENSORS; ++i) {
    a.n[i] = i < m ? lens[i] : 0;
    a.first[i] = i < m ? (unsigned)blocks : ~0u;
    if (i < m) blocks += (lens[i] + ADAMW_TILE - 1) / ADAMW_TILE;
  }
  return blocks;
}

}  // namespace slhip

using namespace slhip;

SLHIP_API int32_t slhip_adamw_step_multi(slhip_ctx* ctx, size_t count, float* const* params, const float* const* grads, float* const* m,
                                         float* const* v, const size_t* lens, float lr, float beta1, float beta2, float eps,
                                         float weight_decay, uint64_t step, uint64_t* step_dev) {
  SLHIP_REQUIRE(ctx && params && grads && m && v && lens, "null argument");
  SLHIP_REQUIRE(count > 0 && count <= ADAMW_MOST, "no tensors, or too many");
  for (size_t i = 0; i < count; ++i) {
    SLHIP_REQUIRE(params[i] && grads[i] && m[i] && v[i] && lens[i] > 0, "null or empty tensor");
    SLHIP_REQUIRE(lens[i] <= ADAMW_LONGEST, "tensor too long");
  }
  const void* const* const arrays[] = {(const void* const*)params, (const void* const*)grads, (const void* const*)m, (const void* const*)v};
  int32_t rc = adamw_overlap("slhip_adamw_step_multi", arrays, 4, 1, count, step_dev, [&](int, size_t i) { return lens[i] * sizeof(float); });
  if (rc) return rc;
  SLHIP_ON_DEVICE(ctx);
  AdamwArgs a;
  rc = adamw_begin(ctx, "slhip_adamw_step_multi", lr, beta1, beta2, eps, weight_decay, step, step_dev, 0, &a.r, &a.step, &a.step_dev);
  if (rc) return rc;
  for (size_t at = 0; at < count; at += ADAMW_TENSORS) {
    const size_t k = count - at < (size_t)ADAMW_TENSORS ? count - at : (size_t)ADAMW_TENSORS;
    for (size_t i = 0; i < (size_t)ADAMW_TENSORS; ++i) {
      const size_t j = at + (i < k ? i : 0);  // no workgroup reads the unused slots
      a.p[i] = params[j]; a.g[i] = grads[j]; a.m[i] = m[j]; a.v[i] = v[j];
    }
    const size_t blocks = adamw_number(a, lens + at, k);
    hipLaunchKernelGGL(adamw_kernel, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, a);
    rc = post_launch();
    if (rc) return rc;
  }
  return SLHIP_OK;
}

SLHIP_API int32_t slhip_adamw8_step_multi(slhip_ctx* ctx, size_t count, float* const* params, const float* const* grads, void* const* m8,
                                          void* const* v8, float* const* scales, const size_t* lens, float lr, float beta1, float beta2,
                                          float eps, float weight_decay, uint64_t step, uint64_t* step_dev, uint64_t seed) {
  SLHIP_REQUIRE(ctx && params && grads && m8 && v8 && scales && lens, "null argument");
  SLHIP_REQUIRE(count > 0 && count <= ADAMW_MOST, "no tensors, or too many");
  for (size_t i = 0; i < count; ++i) {
    SLHIP_REQUIRE(params[i] && grads[i] && m8[i] && v8[i] && scales[i] && lens[i] > 0, "null or empty tensor");
    SLHIP_REQUIRE(lens[i] <= ADAMW_LONGEST, "tensor too long");
    SLHIP_REQUIRE((((uintptr_t)m8[i] | (uintptr_t)v8[i]) & 3) == 0, "8-bit moments must be 4-byte aligned");
  }
  const void* const* const arrays[] = {(const void* const*)params, (const void* const*)grads, (const void* const*)m8, (const void* const*)v8,
                                       (const void* const*)scales};
  int32_t rc = adamw_overlap("slhip_adamw8_step_multi", arrays, 5, 1, count, step_dev, [&](int kind, size_t i) {
    return kind < 2 ? lens[i] * sizeof(float) : kind < 4 ? lens[i] : (lens[i] + ADAMW_BLOCK - 1) / ADAMW_BLOCK * 2 * sizeof(float);
  });
  if (rc) return rc;
  SLHIP_ON_DEVICE(ctx);
  Adamw8Args a;
  rc = adamw_begin(ctx, "slhip_adamw8_step_multi", lr, beta1, beta2, eps, weight_decay, step, step_dev, seed, &a.r, &a.step, &a.step_dev);
  if (rc) return rc;
  for (size_t at = 0; at < count; at += ADAMW_TENSORS) {
    const size_t k = count - at < (size_t)ADAMW_TENSORS ? count - at : (size_t)ADAMW_TENSORS;
    for (size_t i = 0; i < (size_t)ADAMW_TENSORS; ++i) {
      const size_t j = at + (i < k ? i : 0);
      a.p[i] = params[j]; a.g[i] = grads[j]; a.m[i] = (uint8_t*)m8[j]; a.v[i] = (uint8_t*)v8[j]; a.scales[i] = scales[j];
    }
    a.ordinal = (unsigned)at;
    const size_t blocks = adamw_number(a, lens + at, k);
    hipLaunchKernelGGL(adamw8_kernel, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, a);
    rc = post_launch();
    if (rc) return rc;
  }
  return SLHIP_OK;
}
