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
// HBM is the bound: 12 bytes an element forward, 20 (linear) or 24 (sigmoid) backward.  Measured on inputs that change from call
// to call and exceed the last-level cache together, as all figures below unless they say otherwise: 32 x 1000 x 1024 forward 73 us (5.4
// TB/s), backward 147 (5.4); 8 x 2048 x 1024 forward 46 us (4.4), backward 88 (4.6); 65536 x 1024 linear 232 us (5.8 TB/s of the 20 bytes
// that its split moves), backward 316; 32 x 1 x 2048, a token, 2.8 us in the kernel.
#include <type_traits>

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

// V neighbouring channels of a lane.  Where the last lanes of a row would reach past its end they move back to its last V
// channels and store only those that no other lane owns (from `skip` on): every load is a whole vector without a branch
// around it - with one the loads of a run waited for each other (4 x 4099 x 1001 backward: 193 us, 100 without).
template <int V>
struct ScanVec {
  float v[V];
};
template <int V>
struct ScanLane {
  size_t c;  // first channel
  int skip;  // of its channels that another lane owns
  __device__ __forceinline__ ScanLane(size_t first, size_t channels)
      : c(first + V <= channels ? first : channels - V), skip(first >= channels ? V : (int)(first - c)) {}
};
template <int V>
__device__ __forceinline__ ScanVec<V> scan_load(const float* p) {
  ScanVec<V> r;
  if (V == 4) {
    const float4 t = ld4g(p);
    r.v[0] = t.x;
    r.v[V > 1 ? 1 : 0] = t.y;
    r.v[V > 2 ? 2 : 0] = t.z;
    r.v[V > 3 ? 3 : 0] = t.w;
  } else {
    r.v[0] = *p;
  }
  return r;
}
template <int V>
__device__ __forceinline__ ScanVec<V> scan_load_or_zero(const float* p, size_t at) {
  if (p) return scan_load<V>(p + at);
  ScanVec<V> r;
#pragma unroll
  for (int k = 0; k < V; ++k) r.v[k] = 0.0f;
  return r;
}
template <int V>
__device__ __forceinline__ void scan_store(float* p, const ScanVec<V>& r, int skip) {
  if (V == 4 && skip == 0) {
    st4s(p, make_float4(r.v[0], r.v[V > 1 ? 1 : 0], r.v[V > 2 ? 2 : 0], r.v[V > 3 ? 3 : 0]));
    return;
  }
#pragma unroll
  for (int k = 0; k < V; ++k)
    if (k >= skip) p[k] = r.v[k];
}

// p = beta * p + r
template <int V>
__device__ __forceinline__ void scan_grad_store(float* p, ScanVec<V> r, int skip, float beta) {
  if (beta != 0.0f) {
    const ScanVec<V> old = scan_load<V>(p);
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = beta * old.v[k] + r.v[k];
  }
  scan_store<V>(p, r, skip);
}

// (the joins of steps are fused multiply-adds: one rounding a step)
template <int MODE>
__device__ __forceinline__ float scan_coefficient(float gate, float x, float& b) {
  if (MODE == SLHIP_SCAN_LINEAR) {
    b = x;
    return gate;
  }
  float s, rest;
  sigmoid_pair(gate, s, rest);
  b = rest * x;
  return s;
}

// One thread follows V channels through all steps, R of them requested at a time.
template <int MODE, int V, int R>
__global__ __launch_bounds__(256) void scan_rows_kernel(ScanArgs a) {
  const size_t per_row = (a.channels + V - 1) / V;
  const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= a.batch * per_row) return;
  const size_t b = id / per_row;
  const ScanLane<V> lane((id - b * per_row) * V, a.channels);
  const size_t c = lane.c;
  const size_t at = b * a.steps * a.channels + c;
  ScanVec<V> h = scan_load_or_zero<V>(a.h0, b * a.channels + c);
  for (size_t t = 0; t < a.steps; t += R) {
    ScanVec<V> g[R], x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const size_t row = t + r < a.steps ? t + r : a.steps - 1;
      g[r] = scan_load<V>(a.gate + at + row * a.channels);
      x[r] = scan_load<V>(a.x + at + row * a.channels);
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
      scan_store<V>(a.h_out + at + (t + r) * a.channels, h, lane.skip);
    }
  }
  if (a.h_last) scan_store<V>(a.h_last + b * a.channels + c, h, lane.skip);
}

template <int MODE, int V, int R>
__global__ __launch_bounds__(256) void scan_rows_grad_kernel(ScanArgs a) {
  const size_t per_row = (a.channels + V - 1) / V;
  const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= a.batch * per_row) return;
  const size_t b = id / per_row;
  const ScanLane<V> lane((id - b * per_row) * V, a.channels);
  const size_t c = lane.c;
  const size_t at = b * a.steps * a.channels + c, state = b * a.channels + c;
  ScanVec<V> G = scan_load_or_zero<V>(a.dh_last, state);
  const ScanVec<V> first = scan_load_or_zero<V>(a.h0, state);
  for (size_t u = 0; u < a.steps; u += R) {
    ScanVec<V> g[R], x[R], before[R], dh[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const size_t row = u + r < a.steps ? a.steps - 1 - (u + r) : 0;
      g[r] = scan_load<V>(a.gate + at + row * a.channels);
      dh[r] = scan_load<V>(a.dh + at + row * a.channels);
      if (MODE == SLHIP_SCAN_SIGMOID) x[r] = scan_load<V>(a.x + at + row * a.channels);
      before[r] = scan_load<V>(a.h + at + (row > 0 ? row - 1 : 0) * a.channels);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (u + r >= a.steps) break;
      const size_t row = at + (a.steps - 1 - (u + r)) * a.channels;
      if (u + r == a.steps - 1) before[r] = first;
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
          sigmoid_pair(g[r].v[k], s, rest);
          dxv.v[k] = d * rest;
          G.v[k] = s * d;
          dg.v[k] = (dxv.v[k] * s) * (before[r].v[k] - x[r].v[k]);
        }
      }
      if (a.dgate) scan_grad_store<V>(a.dgate + row, dg, lane.skip, a.beta);
      if (a.dx) scan_grad_store<V>(a.dx + row, dxv, lane.skip, a.beta);
    }
  }
  if (a.dh0) scan_grad_store<V>(a.dh0 + state, G, lane.skip, a.beta);
}

// ---------------------------------------------------------------- many steps at a time
// A workgroup owns L * V channels and takes NT / L runs of R steps of them at a time, a run to a thread.  A thread
// folds its run to a pair (A, H) - the run takes a state s to A s + H - the pairs are joined across the workgroup, and with
// the state that then reaches its run a thread goes through it again, out of registers.  The next tile's loads are in
// flight meanwhile.  Nothing is read twice.
//
// Where that leaves the chip idle (few channels, many steps) the steps are also split into chunks over workgroups:
// scan_totals_kernel finds every chunk's pair, and each workgroup then joins those before its own.  That reads the
// inputs of the recurrence a second time; the joins go through the workspace.
struct ScanSplit {
  size_t chunk;    // steps of a workgroup
  float* pairs;    // [chunks - 1][batch][2][channels]
  float* h0;       // the initial state as it was before h_last, which may be the same array, is written
  bool by_xcd;     // rows are not whole lines
};

// What a thread holds of a run of R steps.
template <bool GRAD, int MODE, int V, int R>
struct ScanRun {
  ScanVec<V> g[R];
  ScanVec<V> x[GRAD && MODE == SLHIP_SCAN_LINEAR ? 1 : R];
  ScanVec<V> dh[GRAD ? R : 1];
  ScanVec<V> before[GRAD ? R : 1];
};

// Workgroups are dealt out to the 8 XCDs in turn; this numbers them so that each XCD gets a run of consecutive numbers.
// Neighbouring channel tiles then share an L2, and the 128-byte lines that both have a part of are read and written once:
// 64 x 1000 x 100 forward 24 us instead of 30, 4 x 4099 x 1001 forward 69 instead of 75, backward 98 instead of 107.  Where no line is
// shared it gains nothing and costs up to 4 % (65536 x 1024 linear 243 us, 233 without), so it is left out there.
__device__ __forceinline__ unsigned scan_by_xcd(unsigned id, unsigned count) {
  const unsigned x = id & 7, each = count >> 3, more = count & 7;
  return x * each + (x < more ? x : more) + (id >> 3);
}

// Where a thread's channels and its workgroup's chunk of steps lie.  Steps are counted in running order: u = t forward,
// u = steps - 1 - t backward.
template <int V, int L>
struct ScanPlace {
  size_t b, c, u0, u1;
  unsigned chunk;
  int skip;
  __device__ __forceinline__ ScanPlace(const ScanArgs& a, const ScanSplit& s) {
    unsigned id = blockIdx.y * gridDim.x + blockIdx.x;
    if (s.by_xcd) id = scan_by_xcd(id, gridDim.x * gridDim.y);
    chunk = id / gridDim.x;
    const unsigned group = id - chunk * gridDim.x, tiles = (unsigned)((a.channels + L * V - 1) / (L * V));
    b = group / tiles;
    const ScanLane<V> lane(((size_t)(group % tiles) * L + threadIdx.x % L) * V, a.channels);
    c = lane.c;
    skip = lane.skip;
    u0 = chunk * s.chunk;
    u1 = u0 + s.chunk < a.steps ? u0 + s.chunk : a.steps;
  }
};

// Rows of R steps from u on, those at and past `end` replaced by the step before it (they are masked later).  BACK: one
// step earlier in time (backward only), the first step's by itself.
template <bool GRAD, int V, int R, bool BACK = false>
__device__ __forceinline__ void scan_load_rows(ScanVec<V>* out, const float* src, const ScanArgs& a, size_t b, size_t c, size_t u, size_t end) {
  const size_t first = u < end ? u : end - 1, left = end - first;
  const size_t row = GRAD ? a.steps - 1 - first : first;
  const float* at = src + (b * a.steps + row) * a.channels + c;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    size_t o = (size_t)r < left ? (size_t)r : left - 1;
    if (BACK) o = o < row ? o + 1 : row;
    out[r] = scan_load<V>(GRAD ? at - o * a.channels : at + o * a.channels);
  }
}

template <bool GRAD, int MODE, int V, int R>
__device__ __forceinline__ void scan_load_run(ScanRun<GRAD, MODE, V, R>& run, const ScanArgs& a, size_t b, size_t c, size_t u, size_t end) {
  scan_load_rows<GRAD, V, R>(run.g, a.gate, a, b, c, u, end);
  if (!GRAD) {
    scan_load_rows<GRAD, V, R>(run.x, a.x, a, b, c, u, end);
    return;
  }
  scan_load_rows<GRAD, V, GRAD ? R : 1>(run.dh, a.dh, a, b, c, u, end);
  if (MODE == SLHIP_SCAN_SIGMOID)
    scan_load_rows<GRAD, V, GRAD && MODE == SLHIP_SCAN_LINEAR ? 1 : R>(run.x, a.x, a, b, c, u, end);
  scan_load_rows<GRAD, V, GRAD ? R : 1, true>(run.before, a.h, a, b, c, u, end);
}
// Folds R steps from u on into (A, H): coefficients co and inputs in stay for the second pass.  MASKED: steps at and past
// `end` take the state as it is.
template <bool GRAD, int MODE, int V, int R, bool MASKED>
__device__ __forceinline__ void scan_fold(const ScanVec<V>* g, const ScanVec<V>* x, size_t u, size_t end, ScanVec<V>* co, ScanVec<V>* in,
                                          ScanVec<V>& A, ScanVec<V>& H) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool some = !MASKED || u + r < end;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float c, i, rest = 0.0f;
      if (GRAD) {
        c = g[r].v[k];
        if (MODE == SLHIP_SCAN_SIGMOID) sigmoid_pair(g[r].v[k], c, rest);
        c = some ? c : 1.0f;
        i = some ? x[r].v[k] : 0.0f;                 // dh; what enters is c * dh
        H.v[k] = some ? c * (H.v[k] + i) : H.v[k];
        in[r].v[k] = rest;
      } else {
        c = scan_coefficient<MODE>(g[r].v[k], x[r].v[k], i);
        c = some ? c : 1.0f;
        i = some ? i : 0.0f;
        H.v[k] = some ? fmaf(c, H.v[k], i) : H.v[k];
        in[r].v[k] = i;
      }
      co[r].v[k] = c;
      A.v[k] *= c;
    }
  }
}

// Joins the threads' pairs in the order of their runs: replaces (A, H) by the inclusive pairs within the wave and leaves the
// waves' in LDS, `totals`, for after the next barrier.
template <int V, int L>
__device__ __forceinline__ void scan_join_wave(ScanVec<V>& A, ScanVec<V>& H, float (*totals)[2][L * V]) {
  const int lane = threadIdx.x & 63, run = lane / L;
#pragma unroll
  for (int d = 1; d < 64 / L; d *= 2) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float pa = __shfl_up(A.v[k], d * L, WAVE), ph = __shfl_up(H.v[k], d * L, WAVE);
      if (run >= d) {
        H.v[k] = fmaf(A.v[k], ph, H.v[k]);
        A.v[k] *= pa;
      }
    }
  }
  if (run == 64 / L - 1) {
    const int w = threadIdx.x >> 6, l = lane % L;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      totals[w][0][l * V + k] = A.v[k];
      totals[w][1][l * V + k] = H.v[k];
    }
  }
}
// The state that reaches this thread's run; `carry` becomes the state behind all runs of the workgroup.
template <int V, int L, int NW>
__device__ __forceinline__ ScanVec<V> scan_reach(const ScanVec<V>& A, const ScanVec<V>& H, ScanVec<V>& carry,
                                                 const float (*totals)[2][L * V]) {
  const int lane = threadIdx.x & 63, run = lane / L, l = lane % L, wave = threadIdx.x >> 6;
  ScanVec<V> ea, eh, mine = carry;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    ea.v[k] = L < 64 ? __shfl_up(A.v[k], L % 64, WAVE) : 1.0f;
    eh.v[k] = L < 64 ? __shfl_up(H.v[k], L % 64, WAVE) : 0.0f;
    if (run == 0) {
      ea.v[k] = 1.0f;
      eh.v[k] = 0.0f;
    }
  }
#pragma unroll
  for (int w = 0; w < NW; ++w) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (w == wave) mine.v[k] = carry.v[k];
      carry.v[k] = fmaf(totals[w][0][l * V + k], carry.v[k], totals[w][1][l * V + k]);
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) mine.v[k] = fmaf(ea.v[k], mine.v[k], eh.v[k]);
  return mine;
}

template <int V>
__device__ __forceinline__ void scan_identity(ScanVec<V>& A, ScanVec<V>& H) {
#pragma unroll
  for (int k = 0; k < V; ++k) {
    A.v[k] = 1.0f;
    H.v[k] = 0.0f;
  }
}

// The pair of every chunk but the last: a run of consecutive steps to each group of L threads.  (5.9 TB/s at 65536 x 1024; 8
// or 16 rows requested at a time instead of 4 change nothing.)
template <bool GRAD, int MODE, int V, int L, int R, int NT>
__global__ __launch_bounds__(NT) void scan_totals_kernel(ScanArgs a, ScanSplit s) {
  constexpr int NW = NT / 64, RUNS = NT / L;
  __shared__ __attribute__((aligned(16))) float totals[NW][2][L * V];
  const ScanPlace<V, L> p(a, s);
  const unsigned run = threadIdx.x / L;
  const size_t per = ((p.u1 - p.u0 + RUNS - 1) / RUNS + R - 1) / R * R;
  const size_t begin = p.u0 + run * per, end = begin + per < p.u1 ? begin + per : p.u1;
  ScanVec<V> A, H;
  scan_identity(A, H);
  for (size_t u = begin; u < end; u += R) {
    ScanVec<V> g[R], x[R];
    scan_load_rows<GRAD, V, R>(g, a.gate, a, p.b, p.c, u, end);
    scan_load_rows<GRAD, V, R>(x, GRAD ? a.dh : a.x, a, p.b, p.c, u, end);
    if (u + R <= end) scan_fold<GRAD, MODE, V, R, false>(g, x, u, end, g, x, A, H);
    else scan_fold<GRAD, MODE, V, R, true>(g, x, u, end, g, x, A, H);
  }
  scan_join_wave<V, L>(A, H, totals);
  __syncthreads();
  if (threadIdx.x >= L) return;
  scan_identity(A, H);
#pragma unroll
  for (int w = 0; w < NW; ++w) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      H.v[k] = fmaf(totals[w][0][threadIdx.x * V + k], H.v[k], totals[w][1][threadIdx.x * V + k]);
      A.v[k] *= totals[w][0][threadIdx.x * V + k];
    }
  }
  float* o = s.pairs + ((size_t)p.chunk * a.batch + p.b) * 2 * a.channels + p.c;
#pragma unroll
  for (int k = 0; k < V; ++k)
    if (k >= p.skip) {
      o[k] = A.v[k];
      o[a.channels + k] = H.v[k];
      if (!GRAD && p.chunk == 0 && a.h0) s.h0[p.b * a.channels + p.c + k] = a.h0[p.b * a.channels + p.c + k];
    }
}

// Second pass over a run: from the state h that reaches it, its outputs; returns the state behind it.  WHOLE: every step and
// channel of the run is there and every output wanted, so that the stores have no branch around them: loads that are in
// flight can then be waited for by their number, without the stores behind them (gfx9 counts both together).
template <bool GRAD, int MODE, int V, int R, bool WHOLE>
__device__ __forceinline__ ScanVec<V> scan_apply(const ScanArgs& a, const ScanRun<GRAD, MODE, V, R>& now, const ScanVec<V>* co,
                                                 const ScanVec<V>* in, ScanVec<V> h, const ScanVec<V>& h0, size_t b, size_t c, int skip, size_t u,
                                                 size_t end) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (!WHOLE && u + r >= end) break;
    const size_t at = (b * a.steps + (GRAD ? a.steps - 1 - (u + r) : u + r)) * a.channels + c;
    if (!GRAD) {
#pragma unroll
      for (int k = 0; k < V; ++k) h.v[k] = fmaf(co[r].v[k], h.v[k], in[r].v[k]);
      scan_store<V>(a.h_out + at, h, WHOLE ? 0 : skip);
      continue;
    }
    ScanVec<V> dg, dx;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float d = now.dh[GRAD ? r : 0].v[k] + h.v[k];
      const float before = u + r == a.steps - 1 ? h0.v[k] : now.before[GRAD ? r : 0].v[k];
      h.v[k] = co[r].v[k] * d;
      if (MODE == SLHIP_SCAN_LINEAR) {
        dg.v[k] = d * before;
        dx.v[k] = d;
      } else {
        dx.v[k] = d * in[r].v[k];
        dg.v[k] = (dx.v[k] * co[r].v[k]) * (before - now.x[GRAD && MODE == SLHIP_SCAN_LINEAR ? 0 : r].v[k]);
      }
    }
    if (WHOLE) {
      scan_store<V>(a.dgate + at, dg, 0);
      scan_store<V>(a.dx + at, dx, 0);
      continue;
    }
    if (a.dgate) scan_grad_store<V>(a.dgate + at, dg, skip, a.beta);
    if (a.dx) scan_grad_store<V>(a.dx + at, dx, skip, a.beta);
  }
  return h;
}

template <bool GRAD, int MODE, int V, int L, int R, int NT>
__global__ __launch_bounds__(NT) void scan_tile_kernel(ScanArgs a, ScanSplit s) {
  constexpr int NW = NT / 64, TILE = NT / L * R;
  __shared__ __attribute__((aligned(16))) float totals[2][NW][2][L * V];  // two tiles' in turn: one barrier a tile
  const ScanPlace<V, L> p(a, s);
  const unsigned run = threadIdx.x / L;
  const size_t state = p.b * a.channels + p.c;
  ScanVec<V> A, H, carry = scan_load_or_zero<V>(GRAD ? a.dh_last : gridDim.y > 1 && a.h0 ? s.h0 : a.h0, state);
  const ScanVec<V> h0 = scan_load_or_zero<V>(GRAD ? a.h0 : nullptr, state);
  int buf = 0;
  if (p.chunk > 0) {
    // the chunks before this one: a run of consecutive chunks to each group of L threads
    const unsigned before = p.chunk, per = (before + NT / L - 1) / (NT / L);
    const unsigned q0 = run * per, q1 = q0 + per < before ? q0 + per : before;
    scan_identity(A, H);
    for (unsigned q = q0; q < q1; ++q) {
      const float* o = s.pairs + ((size_t)q * a.batch + p.b) * 2 * a.channels + p.c;
      const ScanVec<V> pa = scan_load<V>(o), ph = scan_load<V>(o + a.channels);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        H.v[k] = fmaf(pa.v[k], H.v[k], ph.v[k]);
        A.v[k] *= pa.v[k];
      }
    }
    scan_join_wave<V, L>(A, H, totals[0]);
    __syncthreads();
    scan_reach<V, L, NW>(A, H, carry, totals[0]);
    buf = 1;
  }
  ScanVec<V> last = carry;
  ScanRun<GRAD, MODE, V, R> next;
  scan_load_run<GRAD, MODE, V, R>(next, a, p.b, p.c, p.u0 + run * R, p.u1);
  auto tile = [&](size_t base, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    const ScanRun<GRAD, MODE, V, R> now = next;
    const size_t u = base + run * R;
    scan_load_run<GRAD, MODE, V, R>(next, a, p.b, p.c, u + TILE, p.u1);  // (behind the last tile: its last row again)
    ScanVec<V> co[R], in[R];
    scan_identity(A, H);
    scan_fold<GRAD, MODE, V, R, !WHOLE>(now.g, GRAD ? now.dh : now.x, u, p.u1, co, in, A, H);
    scan_join_wave<V, L>(A, H, totals[buf]);
    __syncthreads();
    const ScanVec<V> h = scan_reach<V, L, NW>(A, H, carry, totals[buf]);
    last = scan_apply<GRAD, MODE, V, R, WHOLE>(a, now, co, in, h, h0, p.b, p.c, p.skip, u, p.u1);
    buf ^= 1;
  };
  size_t base = p.u0;
  if (__all(p.skip == 0) && (!GRAD || (a.dgate && a.dx && a.beta == 0.0f)))  // (every wave holds all lanes of a run)
    for (; base + TILE <= p.u1; base += TILE) tile(base, std::true_type());
  for (; base < p.u1; base += TILE) tile(base, std::false_type());
  // the state behind the last step is with the thread that took it
  float* const out = GRAD ? a.dh0 : a.h_last;
  if (out && p.u1 == a.steps && run == (a.steps - 1 - p.u0) % TILE / R) {
    if (GRAD) scan_grad_store<V>(out + state, last, p.skip, a.beta);
    else scan_store<V>(out + state, last, p.skip);
  }
}

// ---------------------------------------------------------------- host side
template <bool GRAD, int MODE, int V, int L, int R, int NT>
static int32_t scan_launch_tiles(slhip_ctx* ctx, const ScanArgs& a) {
  constexpr int TILE = NT / L * R;
  const size_t groups = a.batch * ((a.channels + L * V - 1) / (L * V));
  if (groups > MAX_GRID) {
    set_error("slhip_gated_scan: too many channels for one launch");
    return SLHIP_EINVAL;
  }
  const uintptr_t bases = (uintptr_t)a.gate | (uintptr_t)a.x | (uintptr_t)(GRAD ? a.dx : a.h_out);
  ScanSplit s = {a.steps, nullptr, nullptr, a.channels % 32 != 0 || bases % 128 != 0};
  size_t chunks = 1;
  const size_t state = a.batch * a.channels;
  if (groups < (size_t)ctx->num_cu) {
    // two workgroups to a CU, each with a tile at least (65536 x 1024 forward, 8 groups: 64 chunks 232 us, 32 238)
    chunks = ((size_t)ctx->num_cu * 2 + groups - 1) / groups;
    const size_t most = a.steps / TILE;
    if (chunks > most) chunks = most;
    const size_t room = ctx->workspace_bytes / (state * sizeof(float));  // states that the workspace holds
    if (chunks > 1 && 2 * (chunks - 1) + 1 > room) chunks = room > 2 ? (room - 1) / 2 + 1 : 1;
    if (chunks < 1) chunks = 1;
  }
  if (chunks > 1) {
    s.chunk = ((a.steps + chunks - 1) / chunks + TILE - 1) / TILE * TILE;
    chunks = (a.steps + s.chunk - 1) / s.chunk;
  }
  if (chunks > 1) {
    s.h0 = (float*)ctx->workspace;
    s.pairs = s.h0 + state;
    hipLaunchKernelGGL((scan_totals_kernel<GRAD, MODE, V, L, V == 4 ? 4 : 8, NT>), dim3((unsigned)groups, (unsigned)(chunks - 1)), dim3(NT), 0,
                       ctx->stream, a, s);
    const int32_t rc = post_launch();
    if (rc) return rc;
  }
  hipLaunchKernelGGL((scan_tile_kernel<GRAD, MODE, V, L, R, NT>), dim3((unsigned)groups, (unsigned)chunks), dim3(NT), 0, ctx->stream, a, s);
  return post_launch();
}

template <bool GRAD, int MODE>
static int32_t scan_launch(slhip_ctx* ctx, const ScanArgs& a) {
  // steps of a run, and threads: forward longer runs and more of them, backward holds twice the arrays in registers
  // (8 x 2048 x 1024: forward 4 and 512 46.1 us, 4 and 256 48.2, 2 and 512 45.2, which loses where steps are split; backward 2
  // and 256 87.4 us, 2 and 512 89.9, 4 and 256 90.5)
  constexpr int R = GRAD ? 2 : 4, NT = GRAD ? 256 : 512;
  if (a.steps > 8) {
    if (a.channels > 32) {
      // Wide channel tiles, 512 bytes of a row, are what HBM likes best (32 x 1000 x 1024 backward: 146 us at 512 bytes, 167 at
      // 128; forward 73 and 84; 65536 x 1024 linear 232 and 269), if there are enough of them; narrow ones fill the chip where a split of the
      // steps, which reads the inputs of the recurrence twice, would have to otherwise (forward 8 x 2048 x 1024 narrow 46 us, wide and
      // split 68; 4 x 4099 x 1001 has too few narrow tiles too: wide 69, narrow 83, both split; backward 8 x 2048 x 1024 is level).
      const size_t cu = (size_t)ctx->num_cu, wide = a.batch * ((a.channels + 127) / 128), narrow = a.batch * ((a.channels + 31) / 32);
      if (a.channels > 64 && (wide >= cu || narrow < cu || a.steps < 256)) return scan_launch_tiles<GRAD, MODE, 4, 32, R, NT>(ctx, a);
      return scan_launch_tiles<GRAD, MODE, 4, 8, R, NT>(ctx, a);
    }
    if (a.channels > 16) return scan_launch_tiles<GRAD, MODE, 4, 8, R, 256>(ctx, a);
    if (a.channels > 8) return scan_launch_tiles<GRAD, MODE, 4, 4, R, 256>(ctx, a);
    if (a.channels > 3) return scan_launch_tiles<GRAD, MODE, 4, 2, R, 256>(ctx, a);
    if (a.channels > 1) return scan_launch_tiles<GRAD, MODE, 1, 4, 2 * R, 256>(ctx, a);
    return scan_launch_tiles<GRAD, MODE, 1, 1, 2 * R, 256>(ctx, a);
  }
  // a few steps: a thread for each vector of channels
  const int V = a.channels >= 4 ? 4 : 1;
  const size_t threads = a.batch * ((a.channels + V - 1) / V);
  if (!grid_fits(threads, 256)) {
    set_error("slhip_gated_scan: too many channels for one launch");
    return SLHIP_EINVAL;
  }
  const dim3 grid(ceil_div(threads, 256));
  if (GRAD) {
    if (V == 4) hipLaunchKernelGGL((scan_rows_grad_kernel<MODE, 4, 4>), grid, dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((scan_rows_grad_kernel<MODE, 1, 4>), grid, dim3(256), 0, ctx->stream, a);
  } else {
    if (V == 4) hipLaunchKernelGGL((scan_rows_kernel<MODE, 4, 4>), grid, dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((scan_rows_kernel<MODE, 1, 4>), grid, dim3(256), 0, ctx->stream, a);
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
  const Range out = {h, len}, end = {h_last, state};
  if ((h != x && meet(out, {x, len})) || (h != gate && meet(out, {gate, len})) || (!(h == h0 && steps == 1) && meet(out, {h0, state})) ||
      meet(end, out) || meet(end, {x, len}) || meet(end, {gate, len}) || (h_last != h0 && meet(end, {h0, state}))) {
    set_error("slhip_gated_scan: an output overlaps an input, or the other one");
    return SLHIP_EALIAS;
  }
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
  const Range outs[] = {{gate_grad, len}, {x_grad, len}, {h0_grad, state}};
  const Range ins[] = {{gate, len}, {x, len}, {h, len}, {h_grad, len}, {h0, state}, {h_last_grad, state}};
  bool shared = meet(outs[0], outs[1]) || meet(outs[0], outs[2]) || meet(outs[1], outs[2]);
  for (const Range& o : outs)
    for (const Range& i : ins) shared = shared || meet(o, i);
  if (shared) {
    set_error("slhip_gated_scan_grad: a gradient overlaps an input, or another one");
    return SLHIP_EALIAS;
  }
  SLHIP_ON_DEVICE(ctx);
  ScanArgs a = {};
  a.batch = batch; a.steps = steps; a.channels = channels;
  a.gate = gate; a.x = x; a.h0 = h0; a.h = h; a.dh = h_grad; a.dh_last = h_last_grad;
  a.dgate = gate_grad; a.dx = x_grad; a.dh0 = h0_grad; a.beta = beta;
  return mode == SLHIP_SCAN_LINEAR ? scan_launch<true, SLHIP_SCAN_LINEAR>(ctx, a) : scan_launch<true, SLHIP_SCAN_SIGMOID>(ctx, a);
}
