// The gated linear recurrence h_t = a_t * h_{t-1} + b_t along the steps of [batch][steps][channels], and its
// backward pass.
//
//   linear    a = gate                 b = x
//   sigmoid   a = s = 1/(1+exp(-gate)) b = (1 - s) * x
//
// Backward, with d_t the gradient that reaches h_t: d_t = dh_t + a_{t+1} d_{t+1}.  What travels is kept as
// G_t = a_t d_t, so that a step needs its own gate only: d_t = dh_t + G_{t+1}, G_t = a_t d_t - the same recurrence
// run from the last step to the first, with input a_t dh_t.
//
// HBM is the bound: 12 bytes an element forward, 20 (linear) or 24 (sigmoid) backward.
#include "common.hpp"

namespace slhip {

struct ScanArgs {
  size_t batch, steps, channels;
  const float* gate;
  const float* x;
  const float* h0;
  // forward
  float* h_out;
  float* h_last;
  // backward
  const float* h;
  const float* dh;
  const float* dh_last;
  float* dgate;
  float* dx;
  float* dh0;
  float beta;
};

// V neighbouring channels of a lane; the last lane of a row may hold fewer (nv).
template <int V>
struct ScanVec {
  float v[V];
};
template <int V>
__device__ __forceinline__ ScanVec<V> scan_load(const float* p, int nv, float none) {
  ScanVec<V> r;
  if (V == 4 && nv == 4) {
    const float4 t = ld4g(p);
    r.v[0] = t.x;
    r.v[V > 1 ? 1 : 0] = t.y;
    r.v[V > 2 ? 2 : 0] = t.z;
    r.v[V > 3 ? 3 : 0] = t.w;
    return r;
  }
#pragma unroll
  for (int k = 0; k < V; ++k) r.v[k] = k < nv ? p[k] : none;
  return r;
}
template <int V>
__device__ __forceinline__ void scan_store(float* p, const ScanVec<V>& r, int nv) {
  if (V == 4 && nv == 4) {
    st4s(p, make_float4(r.v[0], r.v[V > 1 ? 1 : 0], r.v[V > 2 ? 2 : 0], r.v[V > 3 ? 3 : 0]));
    return;
  }
#pragma unroll
  for (int k = 0; k < V; ++k)
    if (k < nv) p[k] = r.v[k];
}

// s and 1 - s of a sigmoid, each to a few units in its last place at either end: e = exp(-|z|) never
// overflows, and the smaller of the two is e / (1 + e), not a difference.
__device__ __forceinline__ void scan_sigmoid(float z, float& s, float& rest) {
  const float e = expf(-fabsf(z));
  const float big = 1.0f / (1.0f + e), small = e * big;
  s = z >= 0.0f ? big : small;
  rest = z >= 0.0f ? small : big;
  if (z != z) s = rest = z;
}

// (the joins of steps are fused multiply-adds: one rounding a step)
template <int MODE>
__device__ __forceinline__ float scan_coefficient(float gate, float x, float& b) {
  if (MODE == SLHIP_SCAN_LINEAR) {
    b = x;
    return gate;
  }
  float s, rest;
  scan_sigmoid(gate, s, rest);
  b = rest * x;
  return s;
}

// One thread follows V channels through all steps, R of them requested at a time.
template <int MODE, int V, int R>
__global__ __launch_bounds__(256) void scan_rows_kernel(ScanArgs a) {
  const size_t per_row = (a.channels + V - 1) / V;
  const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= a.batch * per_row) return;
  const size_t b = id / per_row, c = (id - b * per_row) * V;
  const int nv = a.channels - c < (size_t)V ? (int)(a.channels - c) : V;
  const size_t at = b * a.steps * a.channels + c;
  ScanVec<V> h;
#pragma unroll
  for (int k = 0; k < V; ++k) h.v[k] = 0.0f;
  if (a.h0) h = scan_load<V>(a.h0 + b * a.channels + c, nv, 0.0f);
  for (size_t t = 0; t < a.steps; t += R) {
    ScanVec<V> g[R], x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const size_t row = t + r < a.steps ? t + r : a.steps - 1;
      g[r] = scan_load<V>(a.gate + at + row * a.channels, nv, 0.0f);
      x[r] = scan_load<V>(a.x + at + row * a.channels, nv, 0.0f);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (t + r >= a.steps) break;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float in;
        const float co = scan_coefficient<MODE>(g[r].v[k], x[r].v[k], in);
        h.v[k] = fmaf(co, h.v[k], in);
      }
      scan_store<V>(a.h_out + at + (t + r) * a.channels, h, nv);
    }
  }
  if (a.h_last) scan_store<V>(a.h_last + b * a.channels + c, h, nv);
}

template <int MODE, int V, int R>
__global__ __launch_bounds__(256) void scan_rows_grad_kernel(ScanArgs a) {
  const size_t per_row = (a.channels + V - 1) / V;
  const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= a.batch * per_row) return;
  const size_t b = id / per_row, c = (id - b * per_row) * V;
  const int nv = a.channels - c < (size_t)V ? (int)(a.channels - c) : V;
  const size_t at = b * a.steps * a.channels + c, state = b * a.channels + c;
  ScanVec<V> G, first;
#pragma unroll
  for (int k = 0; k < V; ++k) G.v[k] = first.v[k] = 0.0f;
  if (a.dh_last) G = scan_load<V>(a.dh_last + state, nv, 0.0f);
  if (a.h0) first = scan_load<V>(a.h0 + state, nv, 0.0f);
  for (size_t u = 0; u < a.steps; u += R) {
    ScanVec<V> g[R], x[R], before[R], dh[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const size_t row = u + r < a.steps ? a.steps - 1 - (u + r) : 0;
      g[r] = scan_load<V>(a.gate + at + row * a.channels, nv, 0.0f);
      dh[r] = scan_load<V>(a.dh + at + row * a.channels, nv, 0.0f);
      if (MODE == SLHIP_SCAN_SIGMOID) x[r] = scan_load<V>(a.x + at + row * a.channels, nv, 0.0f);
      before[r] = first;
      if (row > 0) before[r] = scan_load<V>(a.h + at + (row - 1) * a.channels, nv, 0.0f);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (u + r >= a.steps) break;
      const size_t row = at + (a.steps - 1 - (u + r)) * a.channels;
      ScanVec<V> dg, dxv;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float d = dh[r].v[k] + G.v[k];
        if (MODE == SLHIP_SCAN_LINEAR) {
          dg.v[k] = d * before[r].v[k];
          dxv.v[k] = d;
          G.v[k] = g[r].v[k] * d;
        } else {
          float s, rest;
          scan_sigmoid(g[r].v[k], s, rest);
          dxv.v[k] = d * rest;
          G.v[k] = s * d;
          dg.v[k] = (dxv.v[k] * s) * (before[r].v[k] - x[r].v[k]);
        }
      }
      if (a.dgate) {
        if (a.beta != 0.0f) {
          const ScanVec<V> old = scan_load<V>(a.dgate + row, nv, 0.0f);
#pragma unroll
          for (int k = 0; k < V; ++k) dg.v[k] = a.beta * old.v[k] + dg.v[k];
        }
        scan_store<V>(a.dgate + row, dg, nv);
      }
      if (a.dx) {
        if (a.beta != 0.0f) {
          const ScanVec<V> old = scan_load<V>(a.dx + row, nv, 0.0f);
#pragma unroll
          for (int k = 0; k < V; ++k) dxv.v[k] = a.beta * old.v[k] + dxv.v[k];
        }
        scan_store<V>(a.dx + row, dxv, nv);
      }
    }
  }
  if (a.dh0) {
    if (a.beta != 0.0f) {
      const ScanVec<V> old = scan_load<V>(a.dh0 + state, nv, 0.0f);
#pragma unroll
      for (int k = 0; k < V; ++k) G.v[k] = a.beta * old.v[k] + G.v[k];
    }
    scan_store<V>(a.dh0 + state, G, nv);
  }
}

template <bool GRAD, int MODE>
static int32_t scan_launch(slhip_ctx* ctx, const ScanArgs& a) {
  const int V = a.channels >= 4 ? 4 : 1;
  const size_t threads = a.batch * ((a.channels + V - 1) / V);
  if (!grid_fits(threads, 256)) {
    set_error("slhip_gated_scan: too many channels for one launch");
    return SLHIP_EINVAL;
  }
  const dim3 grid(ceil_div(threads, 256));
  if (GRAD) {
    if (V == 4) hipLaunchKernelGGL((scan_rows_grad_kernel<MODE, 4, 4>), grid, dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((scan_rows_grad_kernel<MODE, 1, 8>), grid, dim3(256), 0, ctx->stream, a);
  } else {
    if (V == 4) hipLaunchKernelGGL((scan_rows_kernel<MODE, 4, 4>), grid, dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((scan_rows_kernel<MODE, 1, 8>), grid, dim3(256), 0, ctx->stream, a);
  }
  return post_launch();
}

}  // namespace slhip

using namespace slhip;

SLHIP_API int32_t slhip_gated_scan(slhip_ctx* ctx, int32_t mode, size_t batch, size_t steps, size_t channels, const float* gate,
                                   const float* x, const float* h0, float* h, float* h_last) {
  size_t state, len;
  SLHIP_REQUIRE(ctx && gate && x && h, "null argument");
  SLHIP_REQUIRE(mode == SLHIP_SCAN_LINEAR || mode == SLHIP_SCAN_SIGMOID, "unknown mode");
  SLHIP_REQUIRE(checked_len(batch, channels, &state) && checked_len(state, steps, &len), "bad dims");
  SLHIP_ON_DEVICE(ctx);
  ScanArgs a = {};
  a.batch = batch; a.steps = steps; a.channels = channels;
  a.gate = gate; a.x = x; a.h0 = h0; a.h_out = h; a.h_last = h_last;
  return mode == SLHIP_SCAN_LINEAR ? scan_launch<false, SLHIP_SCAN_LINEAR>(ctx, a) : scan_launch<false, SLHIP_SCAN_SIGMOID>(ctx, a);
}

SLHIP_API int32_t slhip_gated_scan_grad(slhip_ctx* ctx, int32_t mode, size_t batch, size_t steps, size_t channels, const float* gate,
                                        const float* x, const float* h0, const float* h, float* gate_grad, float* x_grad,
                                        float* h0_grad, const float* h_grad, const float* h_last_grad, float beta) {
  size_t state, len;
  SLHIP_REQUIRE(mode == SLHIP_SCAN_LINEAR || mode == SLHIP_SCAN_SIGMOID, "unknown mode");
  SLHIP_REQUIRE(ctx && gate && h && h_grad && (x || mode == SLHIP_SCAN_LINEAR), "null argument");
  SLHIP_REQUIRE(checked_len(batch, channels, &state) && checked_len(state, steps, &len), "bad dims");
  if (!gate_grad && !x_grad && !h0_grad) return SLHIP_OK;
  SLHIP_ON_DEVICE(ctx);
  ScanArgs a = {};
  a.batch = batch; a.steps = steps; a.channels = channels;
  a.gate = gate; a.x = x; a.h0 = h0; a.h = h; a.dh = h_grad; a.dh_last = h_last_grad;
  a.dgate = gate_grad; a.dx = x_grad; a.dh0 = h0_grad; a.beta = beta;
  return mode == SLHIP_SCAN_LINEAR ? scan_launch<true, SLHIP_SCAN_LINEAR>(ctx, a) : scan_launch<true, SLHIP_SCAN_SIGMOID>(ctx, a);
}
