// Group normalisation with an activation, channels last, and its backward pass.
//
//   mean, rstd = 1/sqrt(var + eps)  over the positions * channels/groups values of a sample's group
//   hat = (x - mean) * rstd         u = hat * weight[c] + bias[c]        out = act(u)
//   g = dout * act'(u), gx = g * weight, < > the mean over the group:
//   dx = rstd * (gx - <gx> - hat * <gx * hat>)       dweight = sum g * hat       dbias = sum g
//
// HBM is the bound: 8 bytes an element forward, 12 backward, if x (and dout) are read once.  Three families of kernels:
//
//   rows     one position a sample (a norm of every row): a row of a group's channels lives in the registers of 4 to 64
//            lanes or of a workgroup, which go on to further rows of the same group with its weights - and, backward,
//            the sums for their gradients - in registers;
//   on chip  all positions of a window of groups fit the registers of a workgroup: x (and dout) are read once;
//   two pass larger ones: a kernel that takes sums, one that applies them.  Runs of positions of a sample go to workgroups
//            of their own, and the second kernel starts where the first one ended, with what the last-level cache still
//            holds.
//
// Measured on inputs that change from call to call and exceed the last-level cache together: 8192 rows x 2048 in 16 groups backward 44
// us (4.6 TB/s), as a layer norm forward 27 (5.0); 32 x 1024 x 512 in 32 groups forward on chip 34 us (4.0 TB/s), backward in two passes
// 67; 32 x 4096 x 512 in two passes forward 131 us (6.1 TB/s of the 12 bytes that those move), backward 243 (5.5 of 20).
//
// In the latter two a window is a run of whole groups, about 32 vectors of channels wide (512 bytes of a row of x): narrower
// pieces of rows than that cost HBM bandwidth.  Groups wider than a workgroup are cut.  A thread keeps to one vector of V
// channels and steps through the positions, so that weights, biases and per-channel sums stay in registers.  V is the
// widest of 4, 2, 1 that divides a group's channels.
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "common.hpp"

namespace slhip {

struct NormArgs {
  size_t N, P, C, G, cg;  // samples, positions, channels, groups, channels of a group
  size_t n0;              // first sample of this launch
  unsigned lanes;         // vectors of channels that a workgroup covers
  unsigned together;      // groups of a window, or 1 where a group is cut into
  unsigned windows;       //   this many windows
  unsigned across;        // windows of a sample
  unsigned rows;          // positions that a workgroup takes at a time
  unsigned chunks;        // runs of positions of a sample, a workgroup each
  size_t chunk;           // positions of a run
  size_t blocks;          // workgroups with work
  bool by_xcd;            // windows share lines with their neighbours
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
  float* cols;            // workspace: [samples * chunks][2][channels], dweight's and dbias's terms
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

// What is left of a normal distribution beyond |u|, erfc(|u| / sqrt 2) / 2, and exp(-u^2 / 2), for x * Phi(x) and its slope.
// erfc(x) is exp(-x^2) times a polynomial without constant in 1/(1 + 0.325 x): the form of Abramowitz and Stegun's formula
// 7.1.26, three terms longer, its coefficients fitted here by reweighted least squares: in exact arithmetic 2.1e-8 off, and
// 2.7e-7 of itself far out.  In 32 bits it is 1.9e-7 off near zero, and far out the rounding of the exponent's argument is what is
// left: 4.6e-7 of itself at |u| = 2, 2.9e-6 at 8, 7e-6 at 12.  From |u| = 13.2 on, where exp(-u^2 / 2) leaves the normal floats, both are
// zero.  (The library's erff takes a branch each for small and large arguments, which both run in a wave; with it the
// arithmetic, not HBM, bounded these kernels: 10 x 961 x 390 forward 17 us.)
__device__ __forceinline__ float norm_tail(float u, float& e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.2298097014427185f, fabsf(u), 1.0f));
  e = __builtin_amdgcn_exp2f(u * u * -0.72134752044448170f);
  float y = fmaf(-0.07500825077295303f, t, 0.27410462498664856f);
  y = fmaf(y, t, -0.24318988621234894f);
  y = fmaf(y, t, 0.2603398561477661f);
  y = fmaf(y, t, -0.003885662415996194f);
  y = fmaf(y, t, 0.10684099793434143f);
  y = fmaf(y, t, 0.08896125853061676f);
  y = fmaf(y, t, 0.09183704107999802f);
  return (y * t) * e;
}

template <int ACT>
__device__ __forceinline__ float norm_act(float u) {
  if (ACT == SLHIP_ACT_RELU) return (u >= 0.0f ? 1.0f : 0.0f) * u;
  if (ACT == SLHIP_ACT_SILU) {
    float q, rest;
    sigmoid_pair(u, q, rest);
    return u * q;
  }
  if (ACT == SLHIP_ACT_GELU) {  // u (1 - tail) or u tail: max(u, 0) - |u| tail; the tail is zero long before 64
    float e;
    return fmaf(-fminf(fabsf(u), 64.0f), norm_tail(u, e), fmaxf(u, 0.0f));
  }
  return u;
}
template <int ACT>
__device__ __forceinline__ float norm_act_grad(float u) {
  if (ACT == SLHIP_ACT_RELU) return u >= 0.0f ? 1.0f : 0.0f;
  if (ACT == SLHIP_ACT_SILU) {
    float q, rest;
    sigmoid_pair(u, q, rest);
    return q * (1.0f + u * rest);
  }
  if (ACT == SLHIP_ACT_GELU) {
    float e;
    const float y = norm_tail(u, e);
    return fmaf(u * 0.39894228040143268f, e, u >= 0.0f ? 1.0f - y : y);
  }
  return 1.0f;
}
// One element of either direction.
template <int ACT>
__device__ __forceinline__ float norm_out(float x, float mean, float rstd, float w, float b) {
  return norm_act<ACT>(fmaf((x - mean) * rstd, w, b));
}
template <int ACT>
__device__ __forceinline__ float norm_upstream(float x, float g, float mean, float rstd, float w, float b, float& hat) {
  hat = (x - mean) * rstd;
  return g * norm_act_grad<ACT>(fmaf(hat, w, b));
}

// Where a workgroup works.  Its number walks the windows fastest, and numbers are dealt out so that an XCD gets a contiguous
// run of them: the 128-byte lines that neighbouring windows share then meet in one L2.
struct NormPlace {
  bool some;          // the workgroup has work
  size_t n, g;        // sample, this thread's group
  unsigned part;      // of the group: window and run of positions
  unsigned local;     // this thread's group within the window
  size_t c;           // its first channel
  size_t first, end;  // its first position, and the end of the workgroup's run
  unsigned lane, row; // its place in the window and among the positions taken at a time
  bool active;
};
template <int V, int NT>
__device__ __forceinline__ NormPlace norm_place(const NormArgs& a, bool backwards) {
  NormPlace p;
  const unsigned blocks = (unsigned)a.blocks, per = (blocks + 7) / 8;
  unsigned id = blockIdx.x;
  p.some = id < blocks;
  if (a.by_xcd) {
    id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    p.some = (blockIdx.x >> 3) < per && id < blocks;
  }
  if (!p.some) id = 0;
  if (backwards) id = blocks - 1 - id;
  const unsigned cgv = (unsigned)(a.cg / V);
  p.lane = threadIdx.x % a.lanes;
  p.row = threadIdx.x / a.lanes;
  const unsigned window = id % a.across;
  id /= a.across;
  const unsigned chunk = id % a.chunks;
  p.n = a.n0 + id / a.chunks;
  p.active = p.some && p.row < a.rows;
  unsigned v;
  if (a.windows > 1) {
    const unsigned piece = window % a.windows, group = window / a.windows;
    p.g = group;
    p.local = 0;
    p.part = chunk * a.windows + piece;
    v = piece * a.lanes + p.lane;
    p.active = p.active && v < cgv;
    p.c = group * a.cg + (size_t)(v < cgv ? v : 0) * V;
  } else {
    p.local = p.lane / cgv;
    v = window * a.together + p.local;  // the group
    p.part = chunk;
    p.active = p.active && v < a.G;
    p.g = v < a.G ? v : a.G - 1;
    p.c = v < a.G ? ((size_t)window * a.lanes + p.lane) * V : 0;
  }
  const size_t begin = (size_t)chunk * a.chunk;
  p.end = begin + a.chunk < a.P ? begin + a.chunk : a.P;
  p.first = begin + p.row;
  if (!p.active) p.first = p.end;
  return p;
}

// Values of a part of a group.
template <int V>
__device__ __forceinline__ float norm_count(const NormArgs& a, unsigned part) {
  const unsigned piece = part % a.windows, chunk = part / a.windows;
  const size_t begin = (size_t)chunk * a.chunk, end = begin + a.chunk < a.P ? begin + a.chunk : a.P;
  const size_t cgv = a.cg / V, v0 = (size_t)piece * a.lanes, v1 = a.windows > 1 && v0 + a.lanes < cgv ? v0 + a.lanes : cgv;
  return (float)((end - begin) * (v1 - v0) * V);
}

// Sums of two values over the threads of each group of the window, in a fixed order: a wave takes the threads of one group
// at a time, or, where there is one group only, its own, and then the waves are added up.  Threads without work bring
// zeros.
template <int NT>
struct NormSums {
  float2 value[NT];
  float2 total[64];
  float reference[64];
};
template <int V, int NT>
__device__ __forceinline__ float2 norm_group_sums(const NormArgs& a, const NormPlace& p, float x, float y, NormSums<NT>& s) {
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float2 t = p.active ? make_float2(x, y) : make_float2(0.0f, 0.0f);
  if (a.together == 1) {
    t.x = wave_reduce<SumOp>(t.x);
    t.y = wave_reduce<SumOp>(t.y);
    if (lane == 0) s.total[wave] = t;
    __syncthreads();
    t = s.total[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) {
      t.x += s.total[i].x;
      t.y += s.total[i].y;
    }
    return t;
  }
  const unsigned cgv = (unsigned)(a.cg / V);
  s.value[threadIdx.x] = t;
  __syncthreads();
  for (unsigned k = wave; k < a.together; k += NT / 64) {
    t = make_float2(0.0f, 0.0f);
    for (unsigned i = lane; i < a.rows * cgv; i += 64) {
      const unsigned r = i / cgv;
      const float2 v = s.value[r * a.lanes + k * cgv + (i - r * cgv)];
      t.x += v.x;
      t.y += v.y;
    }
    t.x = wave_reduce<SumOp>(t.x);
    t.y = wave_reduce<SumOp>(t.y);
    if (lane == 0) s.total[k] = t;
  }
  __syncthreads();
  return s.total[p.local];
}

// Squared differences from another mean: q of them from one, whose distances from it add up to `sum`, less what a move by `shift` to
// the mean takes off; rounding may not make them negative.  Where the squares pass the largest float they stay infinite in every
// kernel - 1/sqrt(var) is zero then - although the difference is one of infinities; NaN stays NaN.
__device__ __forceinline__ float norm_moved(float q, float sum, float shift) {
  const float rest = q - sum * shift;
  return rest > 0.0f ? rest : q < __builtin_huge_valf() ? 0.0f : q;
}

// A working thread's place among those of its group in the workgroup.
struct NormTeam {
  unsigned rank, size;
};
template <int V>
__device__ __forceinline__ NormTeam norm_team(const NormArgs& a, const NormPlace& p) {
  const unsigned cgv = (unsigned)(a.cg / V);
  // a piece of a group: the lanes that this window really has
  const unsigned piece = a.windows > 1 ? p.part % a.windows : 0;
  const unsigned mine = a.windows > 1 ? (cgv - piece * a.lanes < a.lanes ? cgv - piece * a.lanes : a.lanes) : cgv;
  const unsigned lane = a.windows > 1 ? p.lane : p.lane - p.local * cgv;
  return NormTeam{p.row * mine + lane, a.rows * mine};
}

// Joins what the threads of a group know of it: `count` values of mean `here` whose squared differences from that add up to
// `spread`.  Means are taken relative to the one of the group's first thread: it is the mean of many values itself, so
// that no single value, however far from the others, stands between the sums and their difference.  (Relative to zero where
// that mean is within two of the thread's standard deviations of it: a small mean keeps its own digits then.)
template <int V, int NT>
__device__ __forceinline__ void norm_join(const NormArgs& a, const NormPlace& p, unsigned rank, float count, float here, float spread, float total,
                                          NormSums<NT>& s, float& mean, float& m2) {
  if (p.active && rank == 0) s.reference[p.local] = here * here * count > 4.0f * spread ? here : 0.0f;
  __syncthreads();
  const float reference = s.reference[p.local], away = here - reference;
  const float2 t = norm_group_sums<V, NT>(a, p, count * away, spread + count * (away * away), s);
  const float shift = t.x / total;
  mean = reference + shift;
  m2 = norm_moved(t.y, t.x, shift);
}

// A thread's positions, several of them requested at a time: 64 bytes of each array, or 32 of narrow vectors.
template <int V, class F>
__device__ __forceinline__ void norm_each(const NormArgs& a, const NormPlace& p, F&& f) {
  constexpr int U = V == 4 ? 4 : 8;
  const size_t step = (size_t)a.rows * a.C;
  size_t at = (p.n * a.P + p.first) * a.C + p.c, r = p.first;
  for (; r + (U - 1) * (size_t)a.rows < p.end; r += U * (size_t)a.rows, at += U * step) f(at, step, std::integral_constant<int, U>());
  for (; r < p.end; r += a.rows, at += step) f(at, step, std::integral_constant<int, 1>());
}

// ---------------------------------------------------------------- two pass
// Mean and sum of squared differences from it of one workgroup's part of each of its groups.  A thread takes those of the
// vectors that it has at a time and joins them to what it has, and threads and parts are joined the same way: neither a
// group far from zero nor one value far from the others costs the variance its digits.
template <int V>
__global__ __launch_bounds__(256) void norm_stats_kernel(NormArgs a) {
  __shared__ NormSums<256> sums;
  const NormPlace p = norm_place<V, 256>(a, false);
  if (!p.some) return;
  float here = 0.0f, spread = 0.0f, count = 0.0f;
  norm_each<V>(a, p, [&](size_t at, size_t step, auto some) {
    constexpr int U = decltype(some)::value;
    NormVec<V> v[U];
#pragma unroll
    for (int i = 0; i < U; ++i) v[i] = norm_load<V>(a.x + at + i * step);
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) s += v[i].v[k];
    const float m = s * (1.0f / (U * V));
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float d = v[i].v[k] - m;
        q = fmaf(d, d, q);
      }
    const float all = count + U * V, away = m - here, part = (U * V) * __builtin_amdgcn_rcpf(all);
    here = fmaf(away, part, here);
    // (the first values of a thread join nothing: the square of their mean may be infinite, and 0 of it no number)
    spread += count > 0.0f ? fmaf(away * away, count * part, q) : q;
    count = all;
  });
  const unsigned rank = norm_team<V>(a, p).rank;
  float mean, m2;
  norm_join<V, 256>(a, p, rank, count, here, spread, norm_count<V>(a, p.part), sums, mean, m2);
  if (p.active && rank == 0) {
    float* o = a.part + 2 * (((p.n - a.n0) * a.G + p.g) * (a.chunks * a.windows) + p.part);
    o[0] = mean;
    o[1] = m2;
  }
}

template <int V, int ACT>
__global__ __launch_bounds__(256) void norm_apply_kernel(NormArgs a) {
  __shared__ NormSums<256> sums;
  const NormPlace p = norm_place<V, 256>(a, true);
  if (!p.some) return;
  // the threads of a group join its parts
  const unsigned parts = a.chunks * a.windows;
  const float* in = a.part + 2 * ((p.n - a.n0) * a.G + p.g) * parts;
  const float total = (float)(a.P * a.cg);
  const NormTeam t = norm_team<V>(a, p);
  const float reference = in[0];
  float s1 = 0.0f, s2 = 0.0f;
  for (unsigned i = t.rank; i < parts; i += t.size) {
    const float count = norm_count<V>(a, i), away = in[2 * i] - reference;
    s1 = fmaf(count, away, s1);
    s2 += fmaf(count, away * away, in[2 * i + 1]);
  }
  const float2 both = norm_group_sums<V, 256>(a, p, s1, s2, sums);
  const float shift = both.x / total, mean = reference + shift;
  const float rstd = 1.0f / sqrtf(norm_moved(both.y, both.x, shift) / total + a.eps);
  if (!p.active) return;
  if (p.part == 0 && t.rank == 0) {
    if (a.mean) a.mean[p.n * a.G + p.g] = mean;
    if (a.rstd) a.rstd[p.n * a.G + p.g] = rstd;
  }
  const NormVec<V> w = norm_param<V>(a.w, p.c, 1.0f), b = norm_param<V>(a.b, p.c, 0.0f);
  norm_each<V>(a, p, [&](size_t at, size_t step, auto some) {
    constexpr int U = decltype(some)::value;
    NormVec<V> v[U];
#pragma unroll
    for (int i = 0; i < U; ++i) v[i] = norm_load<V>(a.x + at + i * step);
#pragma unroll
    for (int i = 0; i < U; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[i].v[k] = norm_out<ACT>(v[i].v[k], mean, rstd, w.v[k], b.v[k]);
      norm_store<V>(a.out + at + i * step, v[i]);
    }
  });
}

// Sums over the positions that the workgroup's threads of one vector of channels took, left with those of row 0: a
// tree over the rows.
template <int V, int NT>
__device__ __forceinline__ void norm_channel_sums(const NormArgs& a, const NormPlace& p, const float* s1, const float* s2,
                                                  float (*sums)[2 * V + 1]) {
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
      for (int k = 0; k < 2 * V; ++k) sums[threadIdx.x][k] += sums[threadIdx.x + half * a.lanes][k];
    }
  }
}
template <int V>
__device__ __forceinline__ void norm_put_columns(const NormArgs& a, const NormPlace& p, const float* sums, size_t row) {
  float* o = a.cols + row * 2 * a.C + p.c;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    o[k] = sums[2 * k + 1];
    o[a.C + k] = sums[2 * k];
  }
}

// Backward, first pass: per channel the sums of g and g * hat over the workgroup's positions, and over a group's channels
// those weighted by the weights.
template <int V, int ACT>
__global__ __launch_bounds__(256) void norm_grad_sums_kernel(NormArgs a) {
  __shared__ NormSums<256> groups;
  __shared__ float sums[256][2 * V + 1];  // (one word more a row: rows start on different banks)
  const NormPlace p = norm_place<V, 256>(a, false);
  if (!p.some) return;
  const float mean = a.mean[p.n * a.G + p.g], rstd = a.rstd[p.n * a.G + p.g];
  const NormVec<V> w = norm_param<V>(a.w, p.c, 1.0f), b = norm_param<V>(a.b, p.c, 0.0f);
  float s1[V], s2[V];
#pragma unroll
  for (int k = 0; k < V; ++k) s1[k] = s2[k] = 0.0f;
  norm_each<V>(a, p, [&](size_t at, size_t step, auto some) {
    constexpr int U = decltype(some)::value;
    NormVec<V> v[U], g[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      v[i] = norm_load<V>(a.x + at + i * step);
      g[i] = norm_load<V>(a.g + at + i * step);
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float hat;
        const float gu = norm_upstream<ACT>(v[i].v[k], g[i].v[k], mean, rstd, w.v[k], b.v[k], hat);
        s1[k] += gu;
        s2[k] = fmaf(gu, hat, s2[k]);
      }
  });
  if (a.cols) {
    norm_channel_sums<V, 256>(a, p, s1, s2, sums);
    if (p.active && p.row == 0) norm_put_columns<V>(a, p, sums[threadIdx.x], (p.n - a.n0) * a.chunks + p.part / a.windows);
  }
  float ga = 0.0f, gb = 0.0f;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    ga = fmaf(w.v[k], s1[k], ga);
    gb = fmaf(w.v[k], s2[k], gb);
  }
  const float2 t = norm_group_sums<V, 256>(a, p, ga, gb, groups);
  if (p.active && norm_team<V>(a, p).rank == 0) {
    float* o = a.part + 2 * (((p.n - a.n0) * a.G + p.g) * (a.chunks * a.windows) + p.part);
    o[0] = t.x;
    o[1] = t.y;
  }
}

template <int V, int ACT>
__global__ __launch_bounds__(256) void norm_grad_apply_kernel(NormArgs a) {
  __shared__ NormSums<256> sums;
  const NormPlace p = norm_place<V, 256>(a, true);
  if (!p.some) return;
  const float mean = a.mean[p.n * a.G + p.g], rstd = a.rstd[p.n * a.G + p.g];
  const unsigned parts = a.chunks * a.windows;
  const float* in = a.part + 2 * ((p.n - a.n0) * a.G + p.g) * parts;
  const float total = (float)(a.P * a.cg);
  float ga = 0.0f, gb = 0.0f;
  const NormTeam t = norm_team<V>(a, p);
  for (unsigned i = t.rank; i < parts; i += t.size) {
    ga += in[2 * i];
    gb += in[2 * i + 1];
  }
  const float2 both = norm_group_sums<V, 256>(a, p, ga, gb, sums);
  if (!p.active) return;
  ga = both.x / total;
  gb = both.y / total;
  const NormVec<V> w = norm_param<V>(a.w, p.c, 1.0f), b = norm_param<V>(a.b, p.c, 0.0f);
  norm_each<V>(a, p, [&](size_t at, size_t step, auto some) {
    constexpr int U = decltype(some)::value;
    NormVec<V> v[U], g[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      v[i] = norm_load<V>(a.x + at + i * step);
      g[i] = norm_load<V>(a.g + at + i * step);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float hat;
        const float gx = norm_upstream<ACT>(v[i].v[k], g[i].v[k], mean, rstd, w.v[k], b.v[k], hat) * w.v[k];
        v[i].v[k] = rstd * (gx - ga - hat * gb);
      }
      if (a.beta != 0.0f) {
        const NormVec<V> old = norm_load<V>(a.dx + at + i * step);
#pragma unroll
        for (int k = 0; k < V; ++k) v[i].v[k] = a.beta * old.v[k] + v[i].v[k];
      }
      norm_store<V>(a.dx + at + i * step, v[i]);
    }
  });
}

// ---------------------------------------------------------------- on chip
// All P <= rows * K positions of a window in the registers of one workgroup: x is read once.
template <int V, int ACT, int NT, int K>
__global__ __launch_bounds__(NT) void norm_chip_kernel(NormArgs a) {
  __shared__ NormSums<NT> sums;
  const NormPlace p = norm_place<V, NT>(a, false);
  if (!p.some) return;
  const size_t base = p.n * a.P * a.C + p.c;
  NormVec<V> v[K];
#pragma unroll
  for (int i = 0; i < K; ++i) {  // (positions past the end: the last one's values, left out below)
    const size_t r = p.row + (size_t)i * a.rows;
    v[i] = norm_load<V>(a.x + base + (r < a.P ? r : a.P - 1) * a.C);
  }
  // the thread's own mean, and its squared differences from that
  const float total = (float)(a.P * a.cg);
  float count = 0.0f, s = 0.0f;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const bool in = p.row + (size_t)i * a.rows < a.P;
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) t += v[i].v[k];
    s += in ? t : 0.0f;
    count += in ? (float)V : 0.0f;
  }
  const float here = count > 0.0f ? s / count : 0.0f;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float d = v[i].v[k] - here;
      t = fmaf(d, d, t);
    }
    s += p.row + (size_t)i * a.rows < a.P ? t : 0.0f;
  }
  const unsigned rank = norm_team<V>(a, p).rank;
  float mean, m2;
  norm_join<V, NT>(a, p, rank, count, here, s, total, sums, mean, m2);
  const float rstd = 1.0f / sqrtf(m2 / total + a.eps);
  if (!p.active) return;
  if (rank == 0) {
    if (a.mean) a.mean[p.n * a.G + p.g] = mean;
    if (a.rstd) a.rstd[p.n * a.G + p.g] = rstd;
  }
  const NormVec<V> w = norm_param<V>(a.w, p.c, 1.0f), b = norm_param<V>(a.b, p.c, 0.0f);
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const size_t r = p.row + (size_t)i * a.rows;
    if (r >= a.P) break;
#pragma unroll
    for (int k = 0; k < V; ++k) v[i].v[k] = norm_out<ACT>(v[i].v[k], mean, rstd, w.v[k], b.v[k]);
    norm_store<V>(a.out + base + r * a.C, v[i]);
  }
}

template <int V, int ACT, int NT, int K>
__global__ __launch_bounds__(NT) void norm_chip_grad_kernel(NormArgs a) {
  __shared__ NormSums<NT> groups;
  __shared__ float sums[NT][2 * V + 1];
  const NormPlace p = norm_place<V, NT>(a, false);
  if (!p.some) return;
  const size_t base = p.n * a.P * a.C + p.c;
  NormVec<V> v[K], g[K];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const size_t r = p.row + (size_t)i * a.rows, at = base + (r < a.P ? r : a.P - 1) * a.C;
    v[i] = norm_load<V>(a.x + at);
    g[i] = norm_load<V>(a.g + at);
  }
  const float mean = a.mean[p.n * a.G + p.g], rstd = a.rstd[p.n * a.G + p.g], total = (float)(a.P * a.cg);
  const NormVec<V> w = norm_param<V>(a.w, p.c, 1.0f), b = norm_param<V>(a.b, p.c, 0.0f);
  float s1[V], s2[V];
#pragma unroll
  for (int k = 0; k < V; ++k) s1[k] = s2[k] = 0.0f;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const bool in = p.row + (size_t)i * a.rows < a.P;
#pragma unroll
    for (int k = 0; k < V; ++k) {  // x becomes hat, dout becomes g
      float hat;
      const float gu = norm_upstream<ACT>(v[i].v[k], g[i].v[k], mean, rstd, w.v[k], b.v[k], hat);
      v[i].v[k] = hat;
      g[i].v[k] = gu;
      s1[k] += in ? gu : 0.0f;
      s2[k] = in ? fmaf(gu, hat, s2[k]) : s2[k];
    }
  }
  if (a.cols) {
    norm_channel_sums<V, NT>(a, p, s1, s2, sums);
    if (p.active && p.row == 0) norm_put_columns<V>(a, p, sums[threadIdx.x], p.n - a.n0);
  }
  if (!a.dx) return;
  float ga = 0.0f, gb = 0.0f;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    ga = fmaf(w.v[k], s1[k], ga);
    gb = fmaf(w.v[k], s2[k], gb);
  }
  const float2 t = norm_group_sums<V, NT>(a, p, ga, gb, groups);
  if (!p.active) return;
  ga = t.x / total;
  gb = t.y / total;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const size_t r = p.row + (size_t)i * a.rows;
    if (r >= a.P) break;
    NormVec<V> d;
#pragma unroll
    for (int k = 0; k < V; ++k) d.v[k] = rstd * (g[i].v[k] * w.v[k] - ga - v[i].v[k] * gb);
    if (a.beta != 0.0f) {
      const NormVec<V> old = norm_load<V>(a.dx + base + r * a.C);
#pragma unroll
      for (int k = 0; k < V; ++k) d.v[k] = a.beta * old.v[k] + d.v[k];
    }
    norm_store<V>(a.dx + base + r * a.C, d);
  }
}

// ---------------------------------------------------------------- rows
// One position a sample: samples * groups rows of cg channels, one after the other in memory.  A team of threads - `lanes`
// of a wave (BLOCK false), or the whole workgroup - holds a row, K vectors to a thread, and goes on to the row `teams`
// further: teams is a multiple of the groups, so its group, and with it weights, biases and the columns of their
// gradients, stays the same.
struct NormRows {
  unsigned lanes;
  unsigned used;  // teams of a workgroup: as many as are whole rounds of the groups, if there is one
  unsigned fold;  // teams of each group in a workgroup whose column sums are added up there; 1: every team writes its own
  size_t teams;
};

template <bool BLOCK, int NT>
__device__ __forceinline__ float2 norm_row_sums(float x, float y, unsigned lanes, float2* wave_sums) {
  if (!BLOCK) {
    for (unsigned o = lanes / 2; o > 0; o /= 2) {
      x += __shfl_xor(x, o, WAVE);
      y += __shfl_xor(y, o, WAVE);
    }
    return make_float2(x, y);
  }
  x = wave_reduce<SumOp>(x);
  y = wave_reduce<SumOp>(y);
  __syncthreads();  // the sums of an earlier call have been read
  if ((threadIdx.x & 63) == 0) wave_sums[threadIdx.x >> 6] = make_float2(x, y);
  __syncthreads();
  float2 t = wave_sums[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) {
    t.x += wave_sums[i].x;
    t.y += wave_sums[i].y;
  }
  return t;
}

template <int V, int ACT, int NT, int K, bool BLOCK>
__global__ __launch_bounds__(NT) void norm_rows_kernel(NormArgs a, NormRows t) {
  __shared__ float2 wave_sums[NT / 64];
  const unsigned lanes = BLOCK ? NT : t.lanes, lane = threadIdx.x % lanes, cgv = (unsigned)(a.cg / V);
  const unsigned local = BLOCK ? 0 : threadIdx.x / lanes;
  const size_t team = (size_t)blockIdx.x * t.used + local, rows = a.N * a.G;
  if (local >= t.used || team >= t.teams) return;
  const size_t group = team % a.G;
  size_t at[K];  // of a vector within the row; one past the end stands at the last and is left out
  bool in[K];
  NormVec<V> w[K], b[K];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const unsigned q = lane + i * lanes;
    in[i] = q < cgv;
    at[i] = (size_t)(in[i] ? q : cgv - 1) * V;
    w[i] = norm_param<V>(a.w, group * a.cg + at[i], 1.0f);
    b[i] = norm_param<V>(a.b, group * a.cg + at[i], 0.0f);
  }
  const float total = (float)a.cg;
  for (size_t row = team; row < rows; row += t.teams) {
    NormVec<V> v[K];
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] = norm_load<V>(a.x + row * a.cg + at[i]);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) s += in[i] ? v[i].v[k] : 0.0f;
    const float mean = norm_row_sums<BLOCK, NT>(s, 0.0f, lanes, wave_sums).x / total;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float d = v[i].v[k] - mean;
        s = in[i] ? fmaf(d, d, s) : s;
      }
    const float rstd = 1.0f / sqrtf(norm_row_sums<BLOCK, NT>(s, 0.0f, lanes, wave_sums).x / total + a.eps);
    if (lane == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < K; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[i].v[k] = norm_out<ACT>(v[i].v[k], mean, rstd, w[i].v[k], b[i].v[k]);
      if (in[i]) norm_store<V>(a.out + row * a.cg + at[i], v[i]);
    }
  }
}

template <int V, int ACT, int NT, int K, bool BLOCK>
__global__ __launch_bounds__(NT) void norm_rows_grad_kernel(NormArgs a, NormRows t) {
  __shared__ float2 wave_sums[NT / 64];
  const unsigned lanes = BLOCK ? NT : t.lanes, lane = threadIdx.x % lanes, cgv = (unsigned)(a.cg / V);
  const unsigned local = BLOCK ? 0 : threadIdx.x / lanes;
  const size_t rows = a.N * a.G;
  size_t team = (size_t)blockIdx.x * t.used + local;
  const size_t group = team % a.G;
  if (local >= t.used || team >= t.teams) {
    if (t.fold == 1) return;
    team = rows;  // nothing to take, but there for the tree
  }
  size_t at[K];
  bool in[K];
  NormVec<V> w[K], b[K];
  float s1[K][V], s2[K][V];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const unsigned q = lane + i * lanes;
    in[i] = q < cgv;
    at[i] = (size_t)(in[i] ? q : cgv - 1) * V;
    w[i] = norm_param<V>(a.w, group * a.cg + at[i], 1.0f);
    b[i] = norm_param<V>(a.b, group * a.cg + at[i], 0.0f);
#pragma unroll
    for (int k = 0; k < V; ++k) s1[i][k] = s2[i][k] = 0.0f;
  }
  const float total = (float)a.cg;
  NormVec<V> nv[K], ng[K];
  float nmean = 0.0f, nrstd = 0.0f;
  auto request = [&](size_t row) {  // the next row while this one is computed (behind the last: the last again)
    row = row < rows ? row : rows - 1;
#pragma unroll
    for (int i = 0; i < K; ++i) {
      nv[i] = norm_load<V>(a.x + row * a.cg + at[i]);
      ng[i] = norm_load<V>(a.g + row * a.cg + at[i]);
    }
    nmean = a.mean[row];
    nrstd = a.rstd[row];
  };
  request(team);
  for (size_t row = team; row < rows; row += t.teams) {
    NormVec<V> v[K], g[K];
#pragma unroll
    for (int i = 0; i < K; ++i) {
      v[i] = nv[i];
      g[i] = ng[i];
    }
    const float mean = nmean, rstd = nrstd;
    request(row + t.teams);
    float ga = 0.0f, gb = 0.0f;
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float hat;
        float gu = norm_upstream<ACT>(v[i].v[k], g[i].v[k], mean, rstd, w[i].v[k], b[i].v[k], hat);
        gu = in[i] ? gu : 0.0f;
        s1[i][k] += gu;
        s2[i][k] = fmaf(gu, hat, s2[i][k]);
        const float gx = gu * w[i].v[k];
        ga += gx;
        gb = fmaf(gx, hat, gb);
        v[i].v[k] = hat;
        g[i].v[k] = gx;
      }
    if (!a.dx) continue;
    const float2 sums = norm_row_sums<BLOCK, NT>(ga, gb, lanes, wave_sums);
    ga = sums.x / total;
    gb = sums.y / total;
#pragma unroll
    for (int i = 0; i < K; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[i].v[k] = rstd * (g[i].v[k] - ga - v[i].v[k] * gb);
      if (in[i]) {
        float* const o = a.dx + row * a.cg + at[i];
        if (a.beta != 0.0f) {
          const NormVec<V> old = norm_load<V>(o);
#pragma unroll
          for (int k = 0; k < V; ++k) v[i].v[k] = a.beta * old.v[k] + v[i].v[k];
        }
        norm_store<V>(o, v[i]);
      }
    }
  }
  if (!a.cols) return;
  size_t line = BLOCK || t.fold == 1 ? team / a.G : 0;
  if (!BLOCK && t.fold > 1) {
    // the workgroup's `fold` teams of every group leave one line: a tree over them
    __shared__ float sums[BLOCK ? 1 : NT][2 * K * V + 1];
    const unsigned place = local / (unsigned)a.G, apart = (unsigned)a.G * lanes;
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        sums[threadIdx.x][2 * (i * V + k)] = s1[i][k];
        sums[threadIdx.x][2 * (i * V + k) + 1] = s2[i][k];
      }
    unsigned half = 1;
    while (half < t.fold) half *= 2;
    for (half /= 2; half > 0; half /= 2) {
      __syncthreads();
      if (place < half && place + half < t.fold) {
#pragma unroll
        for (int k = 0; k < 2 * K * V; ++k) sums[threadIdx.x][k] += sums[threadIdx.x + half * apart][k];
      }
    }
    if (place > 0) return;
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        s1[i][k] = sums[threadIdx.x][2 * (i * V + k)];
        s2[i][k] = sums[threadIdx.x][2 * (i * V + k) + 1];
      }
    line = blockIdx.x;
  }
  float* const o = a.cols + line * 2 * a.C + group * a.cg;
#pragma unroll
  for (int i = 0; i < K; ++i)
    if (in[i]) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        o[at[i] + k] = s2[i][k];
        o[a.C + at[i] + k] = s1[i][k];
      }
    }
}

// dweight and dbias: the sums of the 2 * C columns of [rows][2][C].  A workgroup takes 32 columns, eight lanes of four to a
// row, 128 rows at a time, and adds up what its rows' threads have in LDS, a wave to a column.
__global__ __launch_bounds__(1024) void norm_columns_kernel(size_t rows, size_t C, const float* __restrict__ cols, float* dw, float* db,
                                                            float beta) {
  __shared__ float sums[128][33];
  const unsigned lane = threadIdx.x & 7, slot = threadIdx.x >> 3;
  const size_t first = (size_t)blockIdx.x * 32, c = first + 4 * lane, width = 2 * C;
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c + 3 < width) {
#pragma unroll 4
    for (size_t r = slot; r < rows; r += 128) {
      const float4 v = ld4g(cols + r * width + c);
      s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
    }
  } else {
    for (size_t r = slot; r < rows; r += 128)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k < width) s[k] += cols[r * width + c + k];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) sums[slot][4 * lane + k] = s[k];
  __syncthreads();
  const unsigned half = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (unsigned k = 0; k < 2; ++k) {
    const unsigned q = wave + 16 * k;
    const float t = wave_reduce<SumOp>(sums[half][q] + sums[half + 64][q]);
    const size_t at = first + q;
    if (half != 0 || at >= width) continue;
    float* const o = at < C ? dw : db;
    const size_t e = at < C ? at : at - C;
    if (o) o[e] = beta != 0.0f ? beta * o[e] + t : t;
  }
}

// ---------------------------------------------------------------- host side
// Windows of about NORM_WINDOW vectors: whole groups, or pieces of one.
constexpr size_t NORM_WINDOW = 32;
// Whether windows begin or end within a 128-byte line, of which their neighbours have the rest.
static bool norm_lines_shared(const NormArgs& a, int V) {
  if (a.across == 1) return false;
  const uintptr_t bases = (uintptr_t)a.x | (uintptr_t)a.out | (uintptr_t)a.g | (uintptr_t)a.dx;
  return bases % 128 != 0 || a.C % 32 != 0 || a.lanes * (unsigned)V % 32 != 0 || (a.windows > 1 && a.cg % 32 != 0);
}
static void norm_windows(NormArgs& a, int V, unsigned threads) {
  const size_t cgv = a.cg / V;
  a.together = 1;
  a.windows = 1;
  if (cgv > threads) {
    a.windows = (unsigned)((cgv + threads - 1) / threads);
    a.lanes = (unsigned)((cgv + a.windows - 1) / a.windows);
  } else {
    if (cgv < NORM_WINDOW) a.together = (unsigned)(NORM_WINDOW / cgv);
    if (a.together > a.G) a.together = (unsigned)a.G;
    a.lanes = (unsigned)(a.together * cgv);
  }
  a.across = (unsigned)((a.G + a.together - 1) / a.together * a.windows);
  a.rows = threads / a.lanes;
  if (a.rows > a.P) a.rows = (unsigned)a.P;
  a.by_xcd = norm_lines_shared(a, V);
}

// Two pass: runs of positions such that the chip gets about 4096 workgroups and a thread still 8 positions.
static void norm_plan(const slhip_ctx* ctx, NormArgs& a, int V) {
  norm_windows(a, V, 256);
  const size_t groups = a.N * a.across, want = (size_t)ctx->num_cu * 16;
  size_t chunks = (want + groups - 1) / groups;
  const size_t most = (a.P + (size_t)a.rows * 8 - 1) / ((size_t)a.rows * 8);
  if (chunks > most) chunks = most;
  if (chunks > 64) chunks = 64;
  if (chunks < 1) chunks = 1;
  a.chunk = (a.P + chunks - 1) / chunks;
  a.chunks = (unsigned)((a.P + a.chunk - 1) / a.chunk);
}

// On chip: whether a window of whole groups fits a workgroup of `threads` that holds K positions to a thread.  As many groups
// together as fit, up to NORM_WINDOW vectors, but no more than leave a workgroup to every CU.
static bool norm_fits(const slhip_ctx* ctx, NormArgs& a, int V, unsigned threads, unsigned K) {
  const size_t cgv = a.cg / V;
  if (cgv > threads) return false;
  a.windows = a.chunks = 1;
  a.chunk = a.P;
  a.together = cgv < NORM_WINDOW ? (unsigned)(NORM_WINDOW / cgv) : 1;
  if (a.together > a.G) a.together = (unsigned)a.G;
  for (; a.together > 0; --a.together) {
    a.lanes = (unsigned)(a.together * cgv);
    a.rows = threads / a.lanes;
    if (a.rows > a.P) a.rows = (unsigned)a.P;
    a.across = (unsigned)((a.G + a.together - 1) / a.together);
    if ((size_t)a.rows * K >= a.P && (a.together == 1 || a.N * a.across >= (size_t)ctx->num_cu)) break;
  }
  if (a.together == 0) return false;
  // Pieces of rows below 96 bytes cost more than the second reading does, unless all of it stays in the caches (forward at 64 x
  // 2048 x 320 in 32 groups, 40 bytes: 230 us here, 129 in two passes; 10 x 961 x 390 in 13, 120 bytes: 12 and 16; 32 x 1000 x
  // 64 in 8, 32 bytes but 8 MiB in all: 8 and 14).
  a.by_xcd = norm_lines_shared(a, V);
  if (a.across > 1 && a.lanes * (size_t)V < 24 && a.N * a.P * a.C > (size_t(1) << 22)) return false;
  a.blocks = a.N * a.across;
  return true;
}

// Rows: the team of a row - K vectors to each of `lanes` threads, in workgroups of NT - and how many teams.
struct NormTeams {
  NormRows t;
  unsigned threads, K;
  size_t blocks, lines;  // workgroups; lines of column sums that they leave
};
static bool norm_teams(const NormArgs& a, int V, size_t most_vectors, size_t most_blocks, NormTeams* r) {
  const size_t cgv = a.cg / V;
  if (cgv > most_vectors) return false;
  r->K = 2;
  r->threads = 256;
  unsigned lanes = 1;
  if (cgv <= 128) {
    while (lanes * 2 < cgv) lanes *= 2;
  } else if (cgv <= 1024) {
    lanes = 256;
    r->K = cgv <= 256 ? 1 : cgv <= 512 ? 2 : 4;
  } else {
    lanes = r->threads = 1024;
    r->K = cgv <= 2048 ? 2 : 4;
  }
  const size_t in_block = r->threads / lanes, rows = a.N * a.G;
  r->t.lanes = lanes;
  r->t.fold = in_block >= 2 * a.G ? (unsigned)(in_block / a.G) : 1;
  r->t.used = (unsigned)(in_block >= a.G ? in_block / a.G * a.G : in_block);
  if (r->threads == 1024) most_blocks = (most_blocks + 1) / 2;  // (one of them to a CU)
  r->blocks = (rows + r->t.used - 1) / r->t.used;
  if (r->blocks > most_blocks) r->blocks = most_blocks;
  const size_t least = (a.G + r->t.used - 1) / r->t.used;  // a team for every group
  if (r->blocks < least) r->blocks = least;
  if (r->blocks > MAX_GRID) return false;
  r->t.teams = r->blocks * r->t.used / a.G * a.G;
  if (r->t.teams > rows) r->t.teams = rows;  // (a multiple of the groups)
  r->lines = r->t.fold > 1 ? r->blocks : r->t.teams / a.G;
  return true;
}

#define NORM_ROWS(KERNEL, NT, K, BLOCK) \
  hipLaunchKernelGGL((KERNEL<V, ACT, NT, K, BLOCK>), dim3((unsigned)r.blocks), dim3(NT), 0, ctx->stream, a, r.t)
#define NORM_ROWS_ANY(KERNEL, LAST)                               \
  do {                                                            \
    if (r.t.lanes <= 64) NORM_ROWS(KERNEL, 256, 2, false);        \
    else if (r.threads == 256 && r.K == 1) NORM_ROWS(KERNEL, 256, 1, true); \
    else if (r.threads == 256 && r.K == 2) NORM_ROWS(KERNEL, 256, 2, true); \
    else if (r.threads == 256) NORM_ROWS(KERNEL, 256, 4, true);   \
    else if (r.K == 2) NORM_ROWS(KERNEL, 1024, 2, true);          \
    else NORM_ROWS(KERNEL, 1024, LAST, true);                     \
  } while (0)

template <int V, int ACT>
static int32_t norm_forward(slhip_ctx* ctx, NormArgs a) {
  NormTeams r;
  if (a.P == 1 && norm_teams(a, V, 4096, (size_t)ctx->num_cu * 16, &r)) {
    NORM_ROWS_ANY(norm_rows_kernel, 4);
    return post_launch();
  }
  // (a few workgroups that hold a large window each would leave most of the chip idle)
  constexpr unsigned K = V == 4 ? 12 : 16;  // positions of a thread in workgroups of 1024: what 128 registers hold
  for (const auto& size : {std::pair<unsigned, unsigned>{256, 4}, {256, 16}, {1024, K}}) {
    if (!norm_fits(ctx, a, V, size.first, size.second) || a.blocks > MAX_GRID - 8) continue;
    if (size.first == 1024 && a.blocks * 4 < (size_t)ctx->num_cu) continue;
    const dim3 grid((unsigned)((a.blocks + 7) / 8 * 8));
    if (size.first == 1024) hipLaunchKernelGGL((norm_chip_kernel<V, ACT, 1024, K>), grid, dim3(1024), 0, ctx->stream, a);
    else if (size.second == 4) hipLaunchKernelGGL((norm_chip_kernel<V, ACT, 256, 4>), grid, dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((norm_chip_kernel<V, ACT, 256, 16>), grid, dim3(256), 0, ctx->stream, a);
    return post_launch();
  }
  norm_plan(ctx, a, V);
  const size_t blocks = (size_t)a.across * a.chunks;  // workgroups of a sample
  const size_t bytes = a.G * a.windows * a.chunks * 2 * sizeof(float);
  // as many samples at a time as the workspace and a launch hold
  size_t samples = ctx->workspace_bytes / bytes;
  if (samples > (MAX_GRID - 8) / blocks) samples = (MAX_GRID - 8) / blocks;
  if (samples == 0) {
    set_error("slhip_group_norm: workspace too small for %zu groups", a.G);
    return SLHIP_EWORKSPACE;
  }
  a.part = (float*)ctx->workspace;
  for (a.n0 = 0; a.n0 < a.N; a.n0 += samples) {
    const size_t k = a.N - a.n0 < samples ? a.N - a.n0 : samples;
    a.blocks = k * blocks;
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

static int32_t norm_columns(slhip_ctx* ctx, size_t rows, size_t C, const float* cols, float* dw, float* db, float beta) {
  if (!grid_fits(C, 16)) {
    set_error("slhip_group_norm_grad: too many channels for one launch");
    return SLHIP_EINVAL;
  }
  hipLaunchKernelGGL(norm_columns_kernel, dim3(ceil_div(2 * C, 32)), dim3(1024), 0, ctx->stream, rows, C, cols, dw, db, beta);
  return post_launch();
}

template <int V, int ACT>
static int32_t norm_backward(slhip_ctx* ctx, NormArgs a, float* dw, float* db) {
  NormTeams r;
  // two workgroups to a CU: a team then takes many rows, and leaves one row of column sums for all of them
  if (a.P == 1 && norm_teams(a, V, 2048, (size_t)ctx->num_cu * 2, &r) && r.lines <= ctx->workspace_bytes / (2 * a.C * sizeof(float))) {
    a.cols = dw || db ? (float*)ctx->workspace : nullptr;
    NORM_ROWS_ANY(norm_rows_grad_kernel, 2);
    const int32_t rc = post_launch();
    return rc || !a.cols ? rc : norm_columns(ctx, r.lines, a.C, a.cols, dw, db, a.beta);
  }
  constexpr unsigned K = V == 4 ? 6 : 8;
  if (a.N <= ctx->workspace_bytes / (2 * a.C * sizeof(float)))
    for (const auto& size : {std::pair<unsigned, unsigned>{256, 4}, {256, 8}, {1024, K}}) {
      if (!norm_fits(ctx, a, V, size.first, size.second) || a.blocks > MAX_GRID - 8) continue;
      if (size.first == 1024 && a.blocks * 4 < (size_t)ctx->num_cu) continue;
      a.cols = dw || db ? (float*)ctx->workspace : nullptr;
      const dim3 grid((unsigned)((a.blocks + 7) / 8 * 8));
      if (size.first == 1024) hipLaunchKernelGGL((norm_chip_grad_kernel<V, ACT, 1024, K>), grid, dim3(1024), 0, ctx->stream, a);
      else if (size.second == 4) hipLaunchKernelGGL((norm_chip_grad_kernel<V, ACT, 256, 4>), grid, dim3(256), 0, ctx->stream, a);
      else hipLaunchKernelGGL((norm_chip_grad_kernel<V, ACT, 256, 8>), grid, dim3(256), 0, ctx->stream, a);
      const int32_t rc = post_launch();
      return rc || !a.cols ? rc : norm_columns(ctx, a.N, a.C, a.cols, dw, db, a.beta);
    }
  norm_plan(ctx, a, V);
  const size_t blocks = (size_t)a.across * a.chunks, parts = a.G * a.windows * a.chunks * 2;
  const size_t bytes = (parts + (size_t)a.chunks * 2 * a.C) * sizeof(float);
  size_t samples = ctx->workspace_bytes / bytes;
  if (samples > (MAX_GRID - 8) / blocks) samples = (MAX_GRID - 8) / blocks;
  if (samples == 0) {
    set_error("slhip_group_norm_grad: workspace too small for %zu channels", a.C);
    return SLHIP_EWORKSPACE;
  }
  if (samples > a.N) samples = a.N;
  a.part = (float*)ctx->workspace;
  a.cols = dw || db ? a.part + samples * parts : nullptr;
  float beta = a.beta;
  for (a.n0 = 0; a.n0 < a.N; a.n0 += samples) {
    const size_t k = a.N - a.n0 < samples ? a.N - a.n0 : samples;
    a.blocks = k * blocks;
    const dim3 grid((unsigned)((a.blocks + 7) / 8 * 8));
    hipLaunchKernelGGL((norm_grad_sums_kernel<V, ACT>), grid, dim3(256), 0, ctx->stream, a);
    int32_t rc = post_launch();
    if (rc) return rc;
    if (a.dx) {
      hipLaunchKernelGGL((norm_grad_apply_kernel<V, ACT>), grid, dim3(256), 0, ctx->stream, a);
      rc = post_launch();
      if (rc) return rc;
    }
    if (a.cols) {
      rc = norm_columns(ctx, k * a.chunks, a.C, a.cols, dw, db, beta);
      if (rc) return rc;
      beta = 1.0f;  // further samples add to what these left
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
  if (channels > 0x7fffffffu) return false;  // (counts of groups, windows and lanes are 32 bits wide)
  *a = NormArgs{};
  a->N = samples; a->P = positions; a->C = channels; a->G = groups; a->cg = channels / groups;
  return true;
}

// Whether an output shares memory with an input or another output.
template <size_t N>
static bool norm_shared(const Range (&outs)[3], const Range (&ins)[N]) {
  bool shared = meet(outs[0], outs[1]) || meet(outs[0], outs[2]) || meet(outs[1], outs[2]);
  for (const Range& o : outs)
    for (const Range& i : ins) shared = shared || meet(o, i);
  return shared;
}

}  // namespace slhip

using namespace slhip;

SLHIP_API int32_t slhip_group_norm(slhip_ctx* ctx, size_t samples, size_t positions, size_t channels, size_t groups, int32_t act,
                                   float eps, const float* x, const float* weight, const float* bias, float* mean, float* rstd,
                                   float* out) {
  NormArgs a;
  SLHIP_REQUIRE(ctx && x && out, "null argument");
  SLHIP_REQUIRE(norm_dims(samples, positions, channels, groups, &a), "bad dims (channels: at most 2^31 - 1), or groups does not divide channels");
  SLHIP_REQUIRE(act >= SLHIP_ACT_NONE && act <= SLHIP_ACT_GELU, "unknown activation");
  SLHIP_REQUIRE(eps >= 0.0f, "eps must not be negative");
  const size_t len = samples * positions * channels, rows = samples * groups;
  const Range outs[] = {{out, len}, {mean, rows}, {rstd, rows}}, ins[] = {{out == x ? nullptr : x, len}, {weight, channels}, {bias, channels}};
  if (norm_shared(outs, ins) || meet({x, len}, outs[1]) || meet({x, len}, outs[2])) {
    set_error("slhip_group_norm: an output overlaps an input, or another one");
    return SLHIP_EALIAS;
  }
  SLHIP_ON_DEVICE(ctx);
  a.x = x; a.w = weight; a.b = bias; a.mean = mean; a.rstd = rstd; a.out = out; a.eps = eps;
  return norm_dispatch(a.cg, act, [&](auto v, auto f) { return norm_forward<decltype(v)::value, decltype(f)::value>(ctx, a); });
}

SLHIP_API int32_t slhip_group_norm_grad(slhip_ctx* ctx, size_t samples, size_t positions, size_t channels, size_t groups, int32_t act,
                                        const float* x, const float* weight, const float* bias, const float* mean, const float* rstd,
                                        float* x_grad, float* weight_grad, float* bias_grad, const float* out_grad, float beta) {
  NormArgs a;
  SLHIP_REQUIRE(ctx && x && mean && rstd && out_grad, "null argument");
  SLHIP_REQUIRE(norm_dims(samples, positions, channels, groups, &a), "bad dims (channels: at most 2^31 - 1), or groups does not divide channels");
  SLHIP_REQUIRE(act >= SLHIP_ACT_NONE && act <= SLHIP_ACT_GELU, "unknown activation");
  if (!x_grad && !weight_grad && !bias_grad) return SLHIP_OK;
  const size_t len = samples * positions * channels, rows = samples * groups;
  const Range outs[] = {{x_grad, len}, {weight_grad, channels}, {bias_grad, channels}};
  const Range ins[] = {{x, len}, {weight, channels}, {bias, channels}, {mean, rows}, {rstd, rows}, {x_grad == out_grad ? nullptr : out_grad, len}};
  if (norm_shared(outs, ins)) {
    set_error("slhip_group_norm_grad: a gradient overlaps an input, or another one");
    return SLHIP_EALIAS;
  }
  SLHIP_ON_DEVICE(ctx);
  a.x = x; a.w = weight; a.b = bias; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dx = x_grad; a.g = out_grad; a.beta = beta;
  return norm_dispatch(a.cg, act, [&](auto v, auto f) {
    return norm_backward<decltype(v)::value, decltype(f)::value>(ctx, a, weight_grad, bias_grad);
  });
}
