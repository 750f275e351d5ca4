// Group normalisation with an activation, channels last, and its backward pass.
//
//   mean, rstd = 1/sqrt(var + eps)  over the positions * channels/groups values of a sample's group
//   hat = (x - mean) * rstd         u = hat * weight[c] + bias[c]        out = act(u)
//   g = dout * act'(u), gx = g * weight, < > the mean over the group:
//   dx = rstd * (gx - <gx> - hat * <gx * hat>)       dweight = sum g * hat       dbias = sum g
//
// HBM is the bound: 8 bytes an element forward, 12 backward, if x (and dout) are read once.
//
// A workgroup works on one group of one sample: a thread keeps to one vector of V channels of the group
// and steps through the positions, so that weights, biases and the per-channel sums of the backward pass
// stay in its registers.  V is the widest of 4, 2, 1 that divides the group's channels.
#include "common.hpp"

namespace slhip {

struct NormArgs {
  size_t N, P, C, G, cg;  // samples, positions, channels, groups, channels of a group
  size_t n0;              // first sample of this launch
  unsigned wv, windows;   // vectors of a group's channels that a workgroup covers; such windows of a group
  unsigned rows;          // positions that a workgroup takes at a time
  unsigned chunks;        // runs of positions of a sample, a workgroup each
  size_t chunk;           // positions of a run
  size_t blocks;          // workgroups with work
  const float* x;
  const float* w;
  const float* b;
  float* mean;
  float* rstd;
  float* out;
  float eps;
  const float* g;
  float* dx;
  float beta;
  float* part;            // workspace: two floats for every group and workgroup of it
  float* cols;            // workspace: [samples * chunks][2][channels]
};

template <int V>
struct NormVec {
  float v[V];
};
typedef float norm_f2 __attribute__((ext_vector_type(2), aligned(4)));
template <int V>
__device__ __forceinline__ NormVec<V> norm_load(const float* p) {
  NormVec<V> r;
  if (V == 4) {
    const float4 t = ld4g(p);
    r.v[0] = t.x; r.v[V > 1 ? 1 : 0] = t.y; r.v[V > 2 ? 2 : 0] = t.z; r.v[V > 3 ? 3 : 0] = t.w;
  } else if (V == 2) {
    const norm_f2 t = *reinterpret_cast<const norm_f2*>(p);
    r.v[0] = t.x; r.v[V > 1 ? 1 : 0] = t.y;
  } else {
    r.v[0] = *p;
  }
  return r;
}
template <int V>
__device__ __forceinline__ void norm_store(float* p, const NormVec<V>& r) {
  if (V == 4) {
    st4s(p, make_float4(r.v[0], r.v[V > 1 ? 1 : 0], r.v[V > 2 ? 2 : 0], r.v[V > 3 ? 3 : 0]));
  } else if (V == 2) {
    const norm_f2 t = {r.v[0], r.v[V > 1 ? 1 : 0]};
    __builtin_nontemporal_store(t, reinterpret_cast<norm_f2*>(p));
  } else {
    st1s(p, r.v[0]);
  }
}
template <int V>
__device__ __forceinline__ NormVec<V> norm_param(const float* p, size_t c, float none) {
  if (p) return norm_load<V>(p + c);
  NormVec<V> r;
#pragma unroll
  for (int k = 0; k < V; ++k) r.v[k] = none;
  return r;
}

template <int ACT>
__device__ __forceinline__ float norm_act(float u) {
  if (ACT == SLHIP_ACT_RELU) return (u >= 0.0f ? 1.0f : 0.0f) * u;
  if (ACT == SLHIP_ACT_SILU) return u / (1.0f + expf(-u));
  if (ACT == SLHIP_ACT_GELU) return 0.5f * u * (1.0f + erff(u * 0.70710678118654752f));
  return u;
}
template <int ACT>
__device__ __forceinline__ float norm_act_grad(float u) {
  if (ACT == SLHIP_ACT_RELU) return u >= 0.0f ? 1.0f : 0.0f;
  if (ACT == SLHIP_ACT_SILU) {
    const float q = 1.0f / (1.0f + expf(-u));
    return q * (1.0f + u * (1.0f - q));
  }
  if (ACT == SLHIP_ACT_GELU)
    return 0.5f * (1.0f + erff(u * 0.70710678118654752f)) + u * expf(-0.5f * u * u) * 0.39894228040143268f;
  return 1.0f;
}

// Where a workgroup works.  Its number walks the groups fastest, and numbers are dealt out so that an XCD gets a
// contiguous run of them: the 128-byte lines that neighbouring groups share then meet in one L2.
struct NormPlace {
  bool some;        // the workgroup has work
  size_t n, g;      // sample, group
  unsigned part;    // of the group: window and run of positions
  size_t c;         // this thread's first channel
  size_t first, end;  // its first position, and the end of the workgroup's run
  unsigned row;     // its place among the positions taken at a time
  bool active;
};
template <int V>
__device__ __forceinline__ NormPlace norm_place(const NormArgs& a) {
  NormPlace p;
  const size_t per = (a.blocks + 7) / 8;
  size_t id = (size_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
  p.some = (blockIdx.x >> 3) < per && id < a.blocks;
  if (!p.some) id = 0;
  p.g = id % a.G;
  id /= a.G;
  const unsigned window = (unsigned)(id % a.windows);
  id /= a.windows;
  const unsigned chunk = (unsigned)(id % a.chunks);
  p.n = a.n0 + id / a.chunks;
  p.part = chunk * a.windows + window;
  const unsigned cgv = (unsigned)(a.cg / V), lane = threadIdx.x % a.wv;
  const unsigned v = window * a.wv + lane;
  p.row = threadIdx.x / a.wv;
  p.active = p.some && p.row < a.rows && v < cgv;
  p.c = p.g * a.cg + (size_t)(v < cgv ? v : 0) * V;
  const size_t begin = (size_t)chunk * a.chunk;
  p.end = begin + a.chunk < a.P ? begin + a.chunk : a.P;
  p.first = begin + p.row;
  if (!p.active) p.first = p.end;
  return p;
}

// Values of a workgroup's part of its group.
template <int V>
__device__ __forceinline__ float norm_count(const NormArgs& a, unsigned part) {
  const unsigned window = part % a.windows, chunk = part / a.windows;
  const size_t begin = (size_t)chunk * a.chunk, end = begin + a.chunk < a.P ? begin + a.chunk : a.P;
  const size_t cgv = a.cg / V, v0 = (size_t)window * a.wv, v1 = v0 + a.wv < cgv ? v0 + a.wv : cgv;
  return (float)((end - begin) * (v1 - v0) * V);
}

// Mean and sum of squared differences from it of one workgroup's part.  A thread sums differences from the first
// value it meets, and threads and parts are then joined by their means: a group far from zero keeps its variance.
template <int V>
__global__ __launch_bounds__(256) void norm_stats_kernel(NormArgs a) {
  __shared__ float red[4];
  const NormPlace p = norm_place<V>(a);
  if (!p.some) return;
  float s1 = 0.0f, s2 = 0.0f, shift = 0.0f, count = 0.0f;
  const float* at = a.x + (p.n * a.P + p.first) * a.C + p.c;
  if (p.first < p.end) shift = at[0];
#pragma unroll 4
  for (size_t r = p.first; r < p.end; r += a.rows, at += a.rows * a.C) {
    const NormVec<V> v = norm_load<V>(at);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float d = v.v[k] - shift;
      s1 += d;
      s2 = fmaf(d, d, s2);
    }
    count += (float)V;
  }
  const float m = count > 0.0f ? s1 / count : 0.0f;
  const float here = shift + m;                       // the thread's mean
  const float spread = fmaxf(s2 - s1 * m, 0.0f);      // and its sum of squared differences
  const float mean = block_reduce<SumOp>(count * here, red) / norm_count<V>(a, p.part);
  const float away = here - mean;
  const float m2 = block_reduce<SumOp>(spread + count * (away * away), red);
  if (threadIdx.x == 0) {
    float* o = a.part + 2 * (((p.n - a.n0) * a.G + p.g) * (a.chunks * a.windows) + p.part);
    o[0] = mean;
    o[1] = m2;
  }
}

template <int V, int ACT>
__global__ __launch_bounds__(256) void norm_apply_kernel(NormArgs a) {
  __shared__ float red[4];
  const NormPlace p = norm_place<V>(a);
  if (!p.some) return;
  const size_t group = (p.n - a.n0) * a.G + p.g;
  const unsigned parts = a.chunks * a.windows;
  const float* in = a.part + 2 * group * parts;
  const float total = (float)(a.P * a.cg);
  float s = 0.0f;
  for (unsigned i = threadIdx.x; i < parts; i += 256) s += norm_count<V>(a, i) * in[2 * i];
  const float mean = block_reduce<SumOp>(s, red) / total;
  s = 0.0f;
  for (unsigned i = threadIdx.x; i < parts; i += 256) {
    const float away = in[2 * i] - mean;
    s += in[2 * i + 1] + norm_count<V>(a, i) * (away * away);
  }
  const float rstd = 1.0f / sqrtf(block_reduce<SumOp>(s, red) / total + a.eps);
  if (p.part == 0 && threadIdx.x == 0) {
    if (a.mean) a.mean[p.n * a.G + p.g] = mean;
    if (a.rstd) a.rstd[p.n * a.G + p.g] = rstd;
  }
  if (!p.active) return;
  const NormVec<V> w = norm_param<V>(a.w, p.c, 1.0f), b = norm_param<V>(a.b, p.c, 0.0f);
  size_t at = (p.n * a.P + p.first) * a.C + p.c;
#pragma unroll 4
  for (size_t r = p.first; r < p.end; r += a.rows, at += a.rows * a.C) {
    NormVec<V> v = norm_load<V>(a.x + at);
#pragma unroll
    for (int k = 0; k < V; ++k) v.v[k] = norm_act<ACT>(((v.v[k] - mean) * rstd) * w.v[k] + b.v[k]);
    norm_store<V>(a.out + at, v);
  }
}

// Backward, first pass: per channel the sums of g and g * hat over the workgroup's positions, and over its channels
// those weighted by the weights.
template <int V, int ACT>
__global__ __launch_bounds__(256) void norm_grad_sums_kernel(NormArgs a) {
  __shared__ float red[4];
  __shared__ float sums[256][2 * V + 1];  // (one word more a row: rows start on different banks)
  const NormPlace p = norm_place<V>(a);
  if (!p.some) return;
  const float mean = a.mean[p.n * a.G + p.g], rstd = a.rstd[p.n * a.G + p.g];
  const NormVec<V> w = norm_param<V>(a.w, p.c, 1.0f), b = norm_param<V>(a.b, p.c, 0.0f);
  float s1[V], s2[V];
#pragma unroll
  for (int k = 0; k < V; ++k) s1[k] = s2[k] = 0.0f;
  size_t at = (p.n * a.P + p.first) * a.C + p.c;
#pragma unroll 4
  for (size_t r = p.first; r < p.end; r += a.rows, at += a.rows * a.C) {
    const NormVec<V> v = norm_load<V>(a.x + at), g = norm_load<V>(a.g + at);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float hat = (v.v[k] - mean) * rstd;
      const float gu = g.v[k] * norm_act_grad<ACT>(hat * w.v[k] + b.v[k]);
      s1[k] += gu;
      s2[k] = fmaf(gu, hat, s2[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    sums[threadIdx.x][2 * k] = s1[k];
    sums[threadIdx.x][2 * k + 1] = s2[k];
  }
  unsigned half = 1;
  while (half < a.rows) half *= 2;
  for (half /= 2; half > 0; half /= 2) {
    __syncthreads();
    if (p.row < half && p.row + half < a.rows) {
#pragma unroll
      for (int k = 0; k < 2 * V; ++k) sums[threadIdx.x][k] += sums[threadIdx.x + half * a.wv][k];
    }
  }
  const bool mine = p.active && p.row == 0;  // (row 0 holds the totals, which its own threads added last)
  float ga = 0.0f, gb = 0.0f;
  if (mine) {
    float* o = a.cols ? a.cols + (((p.n - a.n0) * a.chunks + p.part / a.windows) * 2) * a.C + p.c : nullptr;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float x = sums[threadIdx.x][2 * k], y = sums[threadIdx.x][2 * k + 1];
      ga = fmaf(w.v[k], x, ga);
      gb = fmaf(w.v[k], y, gb);
      if (o) {
        o[k] = y;
        o[a.C + k] = x;
      }
    }
  }
  ga = block_reduce<SumOp>(ga, red);
  gb = block_reduce<SumOp>(gb, red);
  if (threadIdx.x == 0) {
    float* o = a.part + 2 * (((p.n - a.n0) * a.G + p.g) * (a.chunks * a.windows) + p.part);
    o[0] = ga;
    o[1] = gb;
  }
}

template <int V, int ACT>
__global__ __launch_bounds__(256) void norm_grad_apply_kernel(NormArgs a) {
  __shared__ float red[4];
  const NormPlace p = norm_place<V>(a);
  if (!p.some) return;
  const float mean = a.mean[p.n * a.G + p.g], rstd = a.rstd[p.n * a.G + p.g];
  const unsigned parts = a.chunks * a.windows;
  const float* in = a.part + 2 * ((p.n - a.n0) * a.G + p.g) * parts;
  const float total = (float)(a.P * a.cg);
  float ga = 0.0f, gb = 0.0f;
  for (unsigned i = threadIdx.x; i < parts; i += 256) {
    ga += in[2 * i];
    gb += in[2 * i + 1];
  }
  ga = block_reduce<SumOp>(ga, red) / total;
  gb = block_reduce<SumOp>(gb, red) / total;
  if (!p.active) return;
  const NormVec<V> w = norm_param<V>(a.w, p.c, 1.0f), b = norm_param<V>(a.b, p.c, 0.0f);
  size_t at = (p.n * a.P + p.first) * a.C + p.c;
#pragma unroll 4
  for (size_t r = p.first; r < p.end; r += a.rows, at += a.rows * a.C) {
    const NormVec<V> v = norm_load<V>(a.x + at), g = norm_load<V>(a.g + at);
    NormVec<V> d;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float hat = (v.v[k] - mean) * rstd;
      const float gx = g.v[k] * norm_act_grad<ACT>(hat * w.v[k] + b.v[k]) * w.v[k];
      d.v[k] = rstd * (gx - ga - hat * gb);
    }
    if (a.beta != 0.0f) {
      const NormVec<V> old = norm_load<V>(a.dx + at);
#pragma unroll
      for (int k = 0; k < V; ++k) d.v[k] = a.beta * old.v[k] + d.v[k];
    }
    norm_store<V>(a.dx + at, d);
  }
}

// dweight and dbias: the columns of [rows][2][C] summed, 32 columns to a workgroup, 32 rows at a time.
__global__ __launch_bounds__(1024) void norm_columns_kernel(size_t rows, size_t C, const float* __restrict__ cols, float* dw, float* db,
                                                            float beta) {
  __shared__ float sw[32][33], sb[32][33];
  const unsigned lane = threadIdx.x & 31, slot = threadIdx.x >> 5;
  const size_t c = (size_t)blockIdx.x * 32 + lane;
  float x = 0.0f, y = 0.0f;
  if (c < C) {
#pragma unroll 4
    for (size_t r = slot; r < rows; r += 32) {
      x += cols[2 * r * C + c];
      y += cols[(2 * r + 1) * C + c];
    }
  }
  sw[slot][lane] = x;
  sb[slot][lane] = y;
  __syncthreads();
  if (slot < 2) {
    float s = 0.0f;
    for (int k = 0; k < 32; ++k) s += slot == 0 ? sw[k][lane] : sb[k][lane];
    float* const o = slot == 0 ? dw : db;
    if (c < C && o) o[c] = beta != 0.0f ? beta * o[c] + s : s;
  }
}

// ---------------------------------------------------------------- host side
// Cuts every group into windows of channels (a workgroup holds 256 vectors) and runs of positions, such that the chip
// gets about 2048 workgroups and a thread still 8 positions.
static void norm_plan(const slhip_ctx* ctx, NormArgs& a, int V, size_t samples) {
  const size_t cgv = a.cg / V;
  a.windows = (unsigned)((cgv + 255) / 256);
  a.wv = (unsigned)((cgv + a.windows - 1) / a.windows);
  a.rows = 256 / a.wv;
  if (a.rows > a.P) a.rows = (unsigned)a.P;
  const size_t groups = samples * a.G * a.windows, want = (size_t)ctx->num_cu * 8;
  size_t chunks = (want + groups - 1) / groups;
  const size_t most = (a.P + (size_t)a.rows * 8 - 1) / ((size_t)a.rows * 8);
  if (chunks > most) chunks = most;
  if (chunks > 256) chunks = 256;
  if (chunks < 1) chunks = 1;
  a.chunk = (a.P + chunks - 1) / chunks;
  a.chunks = (unsigned)((a.P + a.chunk - 1) / a.chunk);
}

template <int V, int ACT>
static int32_t norm_forward(slhip_ctx* ctx, NormArgs a) {
  norm_plan(ctx, a, V, a.N);
  const size_t each = a.G * a.windows * a.chunks;  // workgroups of a sample
  // as many samples at a time as the workspace and a launch hold
  size_t samples = ctx->workspace_bytes / (each * 2 * sizeof(float));
  if (samples > (MAX_GRID - 8) / each) samples = (MAX_GRID - 8) / each;
  if (samples == 0) {
    set_error("slhip_group_norm: workspace too small for %zu groups", a.G);
    return SLHIP_EWORKSPACE;
  }
  a.part = (float*)ctx->workspace;
  for (a.n0 = 0; a.n0 < a.N; a.n0 += samples) {
    const size_t k = a.N - a.n0 < samples ? a.N - a.n0 : samples;
    a.blocks = k * each;
    const dim3 grid((unsigned)((a.blocks + 7) / 8 * 8));
    hipLaunchKernelGGL((norm_stats_kernel<V>), grid, dim3(256), 0, ctx->stream, a);
    int32_t rc = post_launch();
    if (rc) return rc;
    hipLaunchKernelGGL((norm_apply_kernel<V, ACT>), grid, dim3(256), 0, ctx->stream, a);
    rc = post_launch();
    if (rc) return rc;
  }
  return SLHIP_OK;
}

template <int V, int ACT>
static int32_t norm_backward(slhip_ctx* ctx, NormArgs a, float* dw, float* db) {
  norm_plan(ctx, a, V, a.N);
  const size_t each = a.G * a.windows * a.chunks;
  const size_t bytes = (each * 2 + (size_t)a.chunks * 2 * a.C) * sizeof(float);
  size_t samples = ctx->workspace_bytes / bytes;
  if (samples > (MAX_GRID - 8) / each) samples = (MAX_GRID - 8) / each;
  if (samples == 0) {
    set_error("slhip_group_norm_grad: workspace too small for %zu channels", a.C);
    return SLHIP_EWORKSPACE;
  }
  if (samples > a.N) samples = a.N;
  a.part = (float*)ctx->workspace;
  a.cols = dw || db ? a.part + samples * each * 2 : nullptr;
  float beta = a.beta;
  for (a.n0 = 0; a.n0 < a.N; a.n0 += samples) {
    const size_t k = a.N - a.n0 < samples ? a.N - a.n0 : samples;
    a.blocks = k * each;
    const dim3 grid((unsigned)((a.blocks + 7) / 8 * 8));
    hipLaunchKernelGGL((norm_grad_sums_kernel<V, ACT>), grid, dim3(256), 0, ctx->stream, a);
    int32_t rc = post_launch();
    if (rc) return rc;
    if (a.cols) {
      if (!grid_fits(a.C, 32)) {
        set_error("slhip_group_norm_grad: too many channels for one launch");
        return SLHIP_EINVAL;
      }
      hipLaunchKernelGGL(norm_columns_kernel, dim3(ceil_div(a.C, 32)), dim3(1024), 0, ctx->stream, k * a.chunks, a.C, (const float*)a.cols,
                         dw, db, beta);
      rc = post_launch();
      if (rc) return rc;
      beta = 1.0f;  // further samples add to what these left
    }
    if (a.dx) {
      hipLaunchKernelGGL((norm_grad_apply_kernel<V, ACT>), grid, dim3(256), 0, ctx->stream, a);
      rc = post_launch();
      if (rc) return rc;
    }
  }
  return SLHIP_OK;
}

// Calls f with the vector width and the activation as constants.
template <int V, class F>
static int32_t norm_with_act(int act, F&& f) {
  using std::integral_constant;
  switch (act) {
    case SLHIP_ACT_RELU: return f(integral_constant<int, V>(), integral_constant<int, SLHIP_ACT_RELU>());
    case SLHIP_ACT_SILU: return f(integral_constant<int, V>(), integral_constant<int, SLHIP_ACT_SILU>());
    case SLHIP_ACT_GELU: return f(integral_constant<int, V>(), integral_constant<int, SLHIP_ACT_GELU>());
    default: return f(integral_constant<int, V>(), integral_constant<int, SLHIP_ACT_NONE>());
  }
}
template <class F>
static int32_t norm_dispatch(size_t cg, int act, F&& f) {
  if (cg % 4 == 0) return norm_with_act<4>(act, f);
  if (cg % 2 == 0) return norm_with_act<2>(act, f);
  return norm_with_act<1>(act, f);
}

static bool norm_dims(size_t samples, size_t positions, size_t channels, size_t groups, NormArgs* a) {
  size_t rows, len;
  if (!checked_len(samples, positions, &rows) || !checked_len(rows, channels, &len)) return false;
  if (groups == 0 || channels % groups != 0) return false;
  *a = NormArgs{};
  a->N = samples; a->P = positions; a->C = channels; a->G = groups; a->cg = channels / groups;
  return true;
}

}  // namespace slhip

using namespace slhip;

SLHIP_API int32_t slhip_group_norm(slhip_ctx* ctx, size_t samples, size_t positions, size_t channels, size_t groups, int32_t act,
                                   float eps, const float* x, const float* weight, const float* bias, float* mean, float* rstd,
                                   float* out) {
  NormArgs a;
  SLHIP_REQUIRE(ctx && x && out, "null argument");
  SLHIP_REQUIRE(norm_dims(samples, positions, channels, groups, &a), "bad dims, or groups does not divide channels");
  SLHIP_REQUIRE(act >= SLHIP_ACT_NONE && act <= SLHIP_ACT_GELU, "unknown activation");
  SLHIP_REQUIRE(eps >= 0.0f, "eps must not be negative");
  SLHIP_ON_DEVICE(ctx);
  a.x = x; a.w = weight; a.b = bias; a.mean = mean; a.rstd = rstd; a.out = out; a.eps = eps;
  return norm_dispatch(a.cg, act, [&](auto v, auto f) { return norm_forward<decltype(v)::value, decltype(f)::value>(ctx, a); });
}

SLHIP_API int32_t slhip_group_norm_grad(slhip_ctx* ctx, size_t samples, size_t positions, size_t channels, size_t groups, int32_t act,
                                        const float* x, const float* weight, const float* bias, const float* mean, const float* rstd,
                                        float* x_grad, float* weight_grad, float* bias_grad, const float* out_grad, float beta) {
  NormArgs a;
  SLHIP_REQUIRE(ctx && x && mean && rstd && out_grad, "null argument");
  SLHIP_REQUIRE(norm_dims(samples, positions, channels, groups, &a), "bad dims, or groups does not divide channels");
  SLHIP_REQUIRE(act >= SLHIP_ACT_NONE && act <= SLHIP_ACT_GELU, "unknown activation");
  if (!x_grad && !weight_grad && !bias_grad) return SLHIP_OK;
  SLHIP_ON_DEVICE(ctx);
  a.x = x; a.w = weight; a.b = bias; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dx = x_grad; a.g = out_grad; a.beta = beta;
  return norm_dispatch(a.cg, act, [&](auto v, auto f) {
    return norm_backward<decltype(v)::value, decltype(f)::value>(ctx, a, weight_grad, bias_grad);
  });
}
