// ppn_scan.hip -- the selective state space scan of a policy's memory: whole windows, their gradients, single rows.
//
//   h[t,d,n] = exp(delta A[d,n]) h[t-1,d,n] + delta B[t,n] x[t,d]      delta = softplus(dt + dt_bias)
//   y[t,d]   = (sum_n C[t,n] h[t,d,n] + D[d] x[t,d]) silu(z[t,d])
//
// Bound by the vector units: every element (environment, row, channel) takes one exponential and three multiply-adds per state,
// against 4 elements moved.  The exponential runs at a quarter of the multiply-add's rate, so 16 states cost 128 slots of 4 clocks a
// wave and row.  Hence: one lane owns one channel with all its states in registers (two or four lanes above 16 and 32 states), nothing
// is exchanged between lanes in the forward pass, and B and C (the same for all lanes of a wave) are read once per wave and 8 rows,
// widened to 32 bits in LDS and broadcast from there.  Workgroups are single waves: no barrier is waited for.
#include "ppn_policy.h"

namespace ppn_policy {
namespace {

constexpr int ROWS = 8;          // rows staged together; also the distance of the checkpoints the backward pass restarts from

// ---- lanes -------------------------------------------------------------------------------------------------------------------------
// NS states per lane, LPC lanes per channel, 64 / LPC channels per wave: lane = part * (64 / LPC) + channel, part p has states p NS ..
template <int NS, int LPC> struct Shape {
  static constexpr int CHANNELS = 64 / LPC, STATES = NS * LPC;
};

template <int PATTERN> __device__ inline float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), PATTERN, 0xf, 0xf, true));
}
constexpr int DPP_ROTATE_8 = 0x128, DPP_MIRROR_8 = 0x141, DPP_SWAP_2 = 0x4e, DPP_SWAP_1 = 0xb1;     // row_ror:8, row_half_mirror, quad_perm 2301, 1032

__device__ inline void swap_halves(float& a, float& b) {          // a = {a low, b low}, b = {a high, b high} of the wave's 32-lane halves
  auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
  a = __builtin_bit_cast(float, (unsigned)r[0]);
  b = __builtin_bit_cast(float, (unsigned)r[1]);
}
__device__ inline void swap_rows(float& a, float& b) {            // the same with the odd 16-lane rows of a and the even ones of b
  auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
  a = __builtin_bit_cast(float, (unsigned)r[0]);
  b = __builtin_bit_cast(float, (unsigned)r[1]);
}

// Sum over the lanes of a channel (they are 64 / LPC apart).
template <int LPC> __device__ inline float sum_parts(float v) {
  if constexpr (LPC >= 2) {
    float w = v;
    swap_halves(v, w);
    v += w;
  }
  if constexpr (LPC >= 4) {
    float w = v;
    swap_rows(v, w);
    v += w;
  }
  return v;
}

// Sums V values over the wave's channels (per part), halving: at each distance a lane keeps one half of the values and passes the other half
// on, so 32 values over 64 lanes cost 31 additions a lane and not 32 * 6.  What lane l ends up with: see owner().
template <int V, int LPC> __device__ inline void sum_channels(float (&v)[V]) {
  constexpr int V16 = LPC >= 2 ? V : V / 2, V8 = LPC >= 4 ? V16 : (V16 > 1 ? V16 / 2 : 1);
  static_assert(V >= 16, "");
  const int lane = threadIdx.x;
  if constexpr (LPC < 2) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      float a = v[i], b = v[i + V / 2];
      swap_halves(a, b);
      v[i] = a + b;
    }
  }
  if constexpr (LPC < 4) {
#pragma unroll
    for (int i = 0; i < V16 / 2; ++i) {
      float a = v[i], b = v[i + V16 / 2];
      swap_rows(a, b);
      v[i] = a + b;
    }
  }
  constexpr int V4 = V8 > 1 ? V8 / 2 : 1, V2 = V4 > 1 ? V4 / 2 : 1, V1 = V2 > 1 ? V2 / 2 : 1;
  const bool b3 = lane & 8, b2 = lane & 4, b1 = lane & 2, b0 = lane & 1;
#define PPN_HALVE(COUNT, BIT, PATTERN)                       \
  if constexpr (COUNT > 1) {                                 \
    _Pragma("unroll") for (int i = 0; i < COUNT / 2; ++i) {  \
      float keep = BIT ? v[i + COUNT / 2] : v[i];            \
      float give = BIT ? v[i] : v[i + COUNT / 2];            \
      v[i] = keep + dpp<PATTERN>(give);                      \
    }                                                        \
  } else {                                                   \
    v[0] += dpp<PATTERN>(v[0]);                              \
  }
  PPN_HALVE(V8, b3, DPP_ROTATE_8)
  PPN_HALVE(V4, b2, DPP_MIRROR_8)
  PPN_HALVE(V2, b1, DPP_SWAP_2)
  PPN_HALVE(V1, b0, DPP_SWAP_1)
#undef PPN_HALVE
}
// How many values a lane has after sum_channels, and which is the first (the others follow).
template <int V, int LPC> struct Kept {
  static constexpr int LEVELS = LPC == 1 ? 6 : LPC == 2 ? 5 : 4;
  static constexpr int COUNT = (V >> LEVELS) > 1 ? (V >> LEVELS) : 1;
  static constexpr int SPARE = V >= (1 << LEVELS) ? 0 : LPC == 1 ? (V == 32 ? 1 : 2) : (V == 16 ? 1 : 0);      // low lane bits that hold copies
  __device__ static bool writes(int lane) { return (lane & ((1 << SPARE) - 1)) == 0; }
  __device__ static int first(int lane) { return ((lane & ((1 << LEVELS) - 1)) >> SPARE) * COUNT; }
};

// ---- staging -----------------------------------------------------------------------------------------------------------------------
// ROWS rows of B (and C) of one environment and group, as 32-bit floats in LDS, zero beyond the last state and the last row.
template <typename T, int STATES, bool WITH_C>
__device__ inline void stage(const ppn_scan_args& a, int64_t b, int64_t g, int64_t t0, int64_t t1, float* sb, float* sc) {
  const T* B = (const T*)a.B + b * a.B_batch + g * a.B_group;
  const T* C = (const T*)a.C + b * a.C_batch + g * a.C_group;
#pragma unroll
  for (int i = 0; i < ROWS * STATES / 64; ++i) {
    const int e = threadIdx.x + 64 * i, j = e / STATES, n = e % STATES;
    const bool in = n < a.states && t0 + j < t1;
    sb[e] = in ? to_float(B[(t0 + j) * a.B_time + n]) : 0.0f;
    if constexpr (WITH_C) sc[e] = in ? to_float(C[(t0 + j) * a.C_time + n]) : 0.0f;
  }
}

template <int NS> __device__ inline void read_states(const float* p, float (&v)[NS]) {
#pragma unroll
  for (int i = 0; i < NS; i += 4) {
    float4 q = *(const float4*)(p + i);
    v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
  }
}

// Bit j: row t0 + j begins an episode.  Wave-uniform.
__device__ inline unsigned starts_of(const ppn_scan_args& a, int64_t b, int64_t t0, int64_t t1) {
  if (!a.starts) return 0;
  const int lane = threadIdx.x;
  const bool s = lane < ROWS && t0 + lane < t1 && a.starts[b * a.starts_batch + (t0 + lane) * a.starts_time] != 0;
  return (unsigned)__ballot(s);
}

struct Place { int64_t b, g, d; bool live; int part; };

// Workgroup x: (environment, group, tile of channels), the tile fastest.  A lane past the last channel works on the last one and writes nothing.
template <int NS, int LPC> __device__ inline Place place(const ppn_scan_args& a, int64_t x) {
  constexpr int CHANNELS = Shape<NS, LPC>::CHANNELS;
  const int64_t wide = a.channels / a.groups, tiles = (wide + CHANNELS - 1) / CHANNELS;
  Place p;
  const int64_t gt = x % (a.groups * tiles);
  p.b = x / (a.groups * tiles);
  p.g = gt / tiles;
  const int64_t c = (gt - p.g * tiles) * CHANNELS + threadIdx.x % CHANNELS;
  p.live = c < wide;
  p.d = p.g * wide + (p.live ? c : wide - 1);
  p.part = threadIdx.x / CHANNELS;
  return p;
}

// Row-major [.. x channels x states] tensors of the caller (A, initial and final states).
template <int NS> __device__ inline void load_states(const float* p, int64_t states, int part, float (&v)[NS]) {
#pragma unroll
  for (int n = 0; n < NS; ++n) v[n] = part * NS + n < states ? p[part * NS + n] : 0.0f;
}
template <int NS> __device__ inline void store_states(float* p, int64_t states, int part, const float (&v)[NS]) {
#pragma unroll
  for (int n = 0; n < NS; ++n)
    if (part * NS + n < states) p[part * NS + n] = v[n];
}
// Workspace states: [.. x states x channels], so that a wave's lanes write next to each other.
template <int NS> __device__ inline void load_plane(const float* p, int64_t states, int64_t channels, int64_t d, int part, float (&v)[NS]) {
#pragma unroll
  for (int n = 0; n < NS; ++n) v[n] = part * NS + n < states ? p[(part * NS + n) * channels + d] : 0.0f;
}
template <int NS> __device__ inline void store_plane(float* p, int64_t states, int64_t channels, int64_t d, int part, const float (&v)[NS]) {
#pragma unroll
  for (int n = 0; n < NS; ++n)
    if (part * NS + n < states) p[(part * NS + n) * channels + d] = v[n];
}

__device__ inline float step_size(float dt, float bias, bool soft) {
  const float v = dt + bias;
  return soft ? softplus(v) : v;
}

// ---- forward -----------------------------------------------------------------------------------------------------------------------
// One wave: 64 / LPC channels of one environment over the rows of one chunk (grid.y chunks of `chunk` rows, a multiple of ROWS).
// SUMMARY: no outputs, only what the chunk does to a state that enters it: its own end state from zero, and the sum of delta (the decay of
// the whole chunk is exp(A sum delta)); -1 stands for a chunk that an episode's start cuts, through which nothing passes.
template <typename T, int NS, int LPC, bool SUMMARY>
__global__ void __launch_bounds__(64) scan_forward(ppn_scan_args a, int64_t chunk, int64_t chunks, const float* entering, float* ends, float* sums) {
  constexpr int STATES = Shape<NS, LPC>::STATES;
  __shared__ __align__(16) float sb[2][ROWS * STATES], sc[2][SUMMARY ? 4 : ROWS * STATES];
  const Place p = place<NS, LPC>(a, blockIdx.x);
  const int64_t k = blockIdx.y, t0 = k * chunk, t1 = t0 + chunk < a.time ? t0 + chunk : a.time;
  const bool writes = p.live && p.part == 0;
  float A2[NS], h[NS];
  load_states<NS>(a.A + p.d * a.states, a.states, p.part, A2);
#pragma unroll
  for (int n = 0; n < NS; ++n) A2[n] *= LOG2E, h[n] = 0.0f;
  if constexpr (!SUMMARY) {
    if (entering) load_plane<NS>(entering + (p.b * chunks + k) * a.states * a.channels, a.states, a.channels, p.d, p.part, h);
    else if (a.initial) load_states<NS>(a.initial + (p.b * a.channels + p.d) * a.states, a.states, p.part, h);
  }
  const float bias = a.dt_bias ? a.dt_bias[p.d] : 0.0f, skip = a.D ? a.D[p.d] : 0.0f;
  const bool soft = a.softplus;
  const T* x = (const T*)a.x + p.b * a.x_batch + p.d;
  const T* dt = (const T*)a.dt + p.b * a.dt_batch + p.d;
  const T* z = a.z && !SUMMARY ? (const T*)a.z + p.b * a.z_batch + p.d : nullptr;
  T* y = (T*)a.y + p.b * a.y_batch + p.d;
  float total = 0.0f;
  bool cut = false;
  int turn = 0;
  for (int64_t t = t0; t < t1; t += ROWS, turn ^= 1) {
    T rx[ROWS], rdt[ROWS], rz[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int64_t at = t + j < t1 ? t + j : t1 - 1;
      rx[j] = x[at * a.x_time];
      rdt[j] = dt[at * a.dt_time];
      if (z) rz[j] = z[at * a.z_time];
    }
    const unsigned begins = starts_of(a, p.b, t, t1);
    stage<T, STATES, !SUMMARY>(a, p.b, p.g, t, t1, sb[turn], sc[turn]);
    __syncthreads();
    if constexpr (!SUMMARY) {
      if (a.checkpoints && p.live) {
        const int64_t marks = (a.time + ROWS - 1) / ROWS;
        store_plane<NS>(a.checkpoints + (p.b * marks + t / ROWS) * a.states * a.channels, a.states, a.channels, p.d, p.part, h);
      }
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      if (t + j >= t1) break;
      const float xv = to_float(rx[j]), delta = step_size(to_float(rdt[j]), bias, soft), dx = delta * xv;
      float bv[NS];
      read_states<NS>(sb[turn] + j * STATES + p.part * NS, bv);
      if ((begins >> j) & 1) {
#pragma unroll
        for (int n = 0; n < NS; ++n) h[n] = dx * bv[n];
        cut = true;
      } else {
#pragma unroll
        for (int n = 0; n < NS; ++n) h[n] = __builtin_amdgcn_exp2f(delta * A2[n]) * h[n] + dx * bv[n];
      }
      total += delta;
      if constexpr (!SUMMARY) {
        float cv[NS], s = 0.0f;
        read_states<NS>(sc[turn] + j * STATES + p.part * NS, cv);
#pragma unroll
        for (int n = 0; n < NS; ++n) s += cv[n] * h[n];
        s = sum_parts<LPC>(s) + skip * xv;
        if (z) {
          const float zv = to_float(rz[j]);
          s *= zv * sigmoid(zv);
        }
        if (writes) y[(t + j) * a.y_time] = (T)s;
      }
    }
  }
  if constexpr (SUMMARY) {
    if (p.live) store_plane<NS>(ends + (p.b * chunks + k) * a.states * a.channels, a.states, a.channels, p.d, p.part, h);
    if (writes) {
      sums[((p.b * chunks + k) * 2 + 0) * a.channels + p.d] = total;
      sums[((p.b * chunks + k) * 2 + 1) * a.channels + p.d] = cut ? 1.0f : 0.0f;
    }
  } else if (p.live && a.final_state && t1 == a.time) {
    store_states<NS>(a.final_state + (p.b * a.channels + p.d) * a.states, a.states, p.part, h);
  }
}

// What enters each chunk, in place of what leaves it (forward: chunk k from k - 1; BACKWARD: adjoints, chunk k from k + 1).
template <bool BACKWARD>
__global__ void __launch_bounds__(256) scan_join(ppn_scan_args a, int64_t chunks, float* ends, const float* sums) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, per = a.states * a.channels;
  if (id >= a.batch * per) return;
  const int64_t b = id / per, rest = id - b * per, n = rest / a.channels, d = rest - n * a.channels;
  const float A2 = a.A[d * a.states + n] * LOG2E;
  const float* outside = BACKWARD ? a.dfinal : a.initial;
  float h = outside ? outside[(b * a.channels + d) * a.states + n] : 0.0f;
  float* p = ends + b * chunks * per + rest;
  const float* s = sums + b * chunks * 2 * a.channels + d;
  constexpr int AHEAD = 8;
  for (int64_t i0 = 0; i0 < chunks; i0 += AHEAD) {
    float own[AHEAD], total[AHEAD], cut[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int64_t i = i0 + j < chunks ? i0 + j : chunks - 1, k = BACKWARD ? chunks - 1 - i : i;
      own[j] = p[k * per];
      total[j] = s[(k * 2) * a.channels];
      cut[j] = s[(k * 2 + 1) * a.channels];
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (i0 + j >= chunks) break;
      const int64_t k = BACKWARD ? chunks - 1 - (i0 + j) : i0 + j;
      p[k * per] = h;
      h = cut[j] != 0.0f ? own[j] : own[j] + __builtin_amdgcn_exp2f(total[j] * A2) * h;
    }
  }
}

// ---- backward ----------------------------------------------------------------------------------------------------------------------
// With u[t] = dy[t] silu(z[t]) and the adjoint e[t] = u[t] C[t] + exp(delta[t+1] A) e[t+1]  (0 across an episode's start):
//   dC[t] = sum_d u[t] h[t]       dB[t] = sum_d e[t] delta[t] x[t]       dx[t] = delta[t] sum_n e[t] B[t] + D u[t]
//   q[t] = e[t] exp(delta[t] A) h[t-1];   ddelta[t] = sum_n q[t] A + x[t] sum_n e[t] B[t];   dA = sum_t q[t] delta[t]
// The rows are taken in blocks of 8 from the last to the first: the states of a block are recomputed from its checkpoint and kept in
// registers (8 x NS), then the block is walked backwards.  The sums over channels (dB, dC) are the wave's part of them, one row of partial
// sums per tile of channels, added up by scan_reduce_rows; dA, dD and ddt_bias stay in registers over all rows and environments of the
// workgroup and leave one row of partial sums each.  Both reductions run in a fixed order.
//
// SUMMARY: only what a chunk adds to the adjoint in front of it, and its sum of delta, for chunks that are worked on at once.
template <typename T, int NS, int LPC, bool SUMMARY>
__global__ void __launch_bounds__(64) scan_backward(ppn_scan_args a, int64_t chunk, int64_t chunks, int64_t share, const float* entering, float* ends, float* sums,
                                                    float* rows_out, float* params_out) {
  constexpr int STATES = Shape<NS, LPC>::STATES, CHANNELS = Shape<NS, LPC>::CHANNELS;
  __shared__ __align__(16) float sb[ROWS * STATES], sc[ROWS * STATES];
  const int64_t wide = a.channels / a.groups, tiles = (wide + CHANNELS - 1) / CHANNELS;
  const int64_t k = blockIdx.y, first = k * chunk, last = first + chunk < a.time ? first + chunk : a.time, marks = (a.time + ROWS - 1) / ROWS;
  const bool soft = a.softplus;
  Place p = place<NS, LPC>(a, blockIdx.x);
  const bool writes = p.live && p.part == 0;
  const float alive = p.live ? 1.0f : 0.0f;
  const int64_t b0 = p.b * share, b1 = b0 + share < a.batch ? b0 + share : a.batch;
  float A2[NS], dA[NS], e[NS];
  load_states<NS>(a.A + p.d * a.states, a.states, p.part, A2);
#pragma unroll
  for (int n = 0; n < NS; ++n) A2[n] *= LOG2E, dA[n] = 0.0f;
  const float bias = a.dt_bias ? a.dt_bias[p.d] : 0.0f, skip = a.D ? a.D[p.d] : 0.0f;
  float dskip = 0.0f, dbias = 0.0f;
  for (int64_t b = b0; b < b1; ++b) {
    const T* x = (const T*)a.x + b * a.x_batch + p.d;
    const T* dt = (const T*)a.dt + b * a.dt_batch + p.d;
    const T* z = a.z ? (const T*)a.z + b * a.z_batch + p.d : nullptr;
    const T* dy = (const T*)a.dy + b * a.dy_batch + p.d;
    T* dx = (T*)a.dx + b * a.dx_batch + p.d;
    T* ddt = (T*)a.ddt + b * a.ddt_batch + p.d;
    T* dz = a.dz ? (T*)a.dz + b * a.dz_batch + p.d : nullptr;
#pragma unroll
    for (int n = 0; n < NS; ++n) e[n] = 0.0f;
    if constexpr (!SUMMARY) {
      if (entering) load_plane<NS>(entering + (b * chunks + k) * a.states * a.channels, a.states, a.channels, p.d, p.part, e);
      else if (a.dfinal) load_states<NS>(a.dfinal + (b * a.channels + p.d) * a.states, a.states, p.part, e);
    }
    float total = 0.0f;
    bool cut = false;
    for (int64_t t = (last - 1) / ROWS * ROWS; t >= first && last > first; t -= ROWS) {
      T rx[ROWS], rdt[ROWS], rz[ROWS], rdy[ROWS];
      float h[SUMMARY ? 1 : ROWS + 1][NS];
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        const int64_t at = t + j < last ? t + j : last - 1;
        if constexpr (!SUMMARY) rx[j] = x[at * a.x_time];
        rdt[j] = dt[at * a.dt_time];
        rdy[j] = dy[at * a.dy_time];
        if (z) rz[j] = z[at * a.z_time];
      }
      if constexpr (!SUMMARY) load_plane<NS>(a.checkpoints + (b * marks + t / ROWS) * a.states * a.channels, a.states, a.channels, p.d, p.part, h[0]);
      const unsigned begins = starts_of(a, b, t, last);
      __syncthreads();
      stage<T, STATES, true>(a, b, p.g, t, last, sb, sc);
      __syncthreads();
      if constexpr (!SUMMARY) {
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          const float delta = step_size(to_float(rdt[j]), bias, soft), w = delta * to_float(rx[j]);
          float bv[NS];
          read_states<NS>(sb + j * STATES + p.part * NS, bv);
          if ((begins >> j) & 1) {
#pragma unroll
            for (int n = 0; n < NS; ++n) h[j + 1][n] = w * bv[n];
          } else {
#pragma unroll
            for (int n = 0; n < NS; ++n) h[j + 1][n] = __builtin_amdgcn_exp2f(delta * A2[n]) * h[j][n] + w * bv[n];
          }
        }
      }
#pragma unroll
      for (int j = ROWS - 1; j >= 0; --j) {
        if (t + j >= last) continue;
        const float raw = to_float(rdt[j]) + bias, delta = soft ? softplus(raw) : raw;
        const float up = to_float(rdy[j]);
        float u = up, sg = 0.0f, zv = 0.0f;
        if (z) {
          zv = to_float(rz[j]);
          sg = sigmoid(zv);
          u = up * zv * sg;
        }
        float cv[NS];
        read_states<NS>(sc + j * STATES + p.part * NS, cv);
        const bool begin = (begins >> j) & 1;
        if constexpr (SUMMARY) {
#pragma unroll
          for (int n = 0; n < NS; ++n) e[n] = begin ? 0.0f : __builtin_amdgcn_exp2f(delta * A2[n]) * (e[n] + u * cv[n]);
          total += delta;
          cut |= begin;
        } else {
          const float xv = to_float(rx[j]), w = delta * xv;
          float bv[NS], sums2[2 * NS], s = 0.0f, through = 0.0f, decay = 0.0f;
          read_states<NS>(sb + j * STATES + p.part * NS, bv);
          const float ul = u * alive, wl = w * alive;        // (a lane past the last channel adds nothing to the sums over channels)
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            s += cv[n] * h[j + 1][n];
            e[n] += u * cv[n];
            sums2[NS + n] = ul * h[j + 1][n];
            sums2[n] = wl * e[n];
            through += e[n] * bv[n];
            if (begin) {
              e[n] = 0.0f;
            } else {
              e[n] *= __builtin_amdgcn_exp2f(delta * A2[n]);
              const float q = e[n] * h[j][n];
              dA[n] += q * delta;
              decay += q * A2[n];
            }
          }
          sum_channels<2 * NS, LPC>(sums2);
          typedef Kept<2 * NS, LPC> K;
          const int lane = threadIdx.x;
          if (K::writes(lane)) {
            const int64_t tile = blockIdx.x % (a.groups * tiles) % tiles;
            float* out = rows_out + (((tile * a.batch + b) * a.time + t + j) * a.groups + p.g) * 2 * a.states;
#pragma unroll
            for (int i = 0; i < K::COUNT; ++i) {
              const int v = K::first(lane) + i, n = p.part * NS + v % NS;
              if (n < a.states) out[(v / NS) * a.states + n] = sums2[i];
            }
          }
          s = sum_parts<LPC>(s) + skip * xv;
          through = sum_parts<LPC>(through);
          decay = sum_parts<LPC>(decay) * (1.0f / LOG2E);
          float dd = decay + through * xv;
          if (soft) dd *= raw > 20.0f ? 1.0f : sigmoid(raw);
          dbias += dd;
          dskip += u * xv;
          if (writes) {
            dx[(t + j) * a.dx_time] = (T)(through * delta + skip * u);
            ddt[(t + j) * a.ddt_time] = (T)dd;
            if (dz) dz[(t + j) * a.dz_time] = (T)(up * s * sg * (1.0f + zv * (1.0f - sg)));
          }
        }
      }
    }
    if constexpr (SUMMARY) {
      if (p.live) store_plane<NS>(ends + (b * chunks + k) * a.states * a.channels, a.states, a.channels, p.d, p.part, e);
      if (writes) {
        sums[((b * chunks + k) * 2 + 0) * a.channels + p.d] = total;
        sums[((b * chunks + k) * 2 + 1) * a.channels + p.d] = cut ? 1.0f : 0.0f;
      }
    } else if (p.live && a.dinitial && first == 0) {
      store_states<NS>(a.dinitial + (b * a.channels + p.d) * a.states, a.states, p.part, e);
    }
  }
  if constexpr (!SUMMARY) {
    float* out = params_out + (p.b * chunks + k) * (a.states + 2) * a.channels;
    if (p.live) store_plane<NS>(out, a.states, a.channels, p.d, p.part, dA);
    if (writes) {
      out[a.states * a.channels + p.d] = dskip;
      out[(a.states + 1) * a.channels + p.d] = dbias;
    }
  }
}

// dB and dC out of the tiles' partial rows [tiles x rows x 2 states].
template <typename T>
__global__ void __launch_bounds__(256) scan_reduce_rows(const float* in, int64_t tiles, int64_t rows, int64_t states, T* dB, T* dC) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, count = rows * 2 * states;
  if (id >= count) return;
  float s = 0.0f;
  for (int64_t t = 0; t < tiles; ++t) s += in[t * count + id];
  const int64_t row = id / (2 * states), v = id - row * 2 * states;
  if (v < states) dB[row * states + v] = (T)s;
  else dC[row * states + v - states] = (T)s;
}

// dA, dD, ddt_bias out of the workgroups' partial rows [shares x (states + 2) x channels].
__global__ void __launch_bounds__(256) scan_reduce_params(const float* in, int64_t shares, int64_t states, int64_t channels, float* dA, float* dD, float* dbias) {
  const int64_t columns = (states + 2) * channels, col = (int64_t)blockIdx.x * 32 + threadIdx.x % 32;
  const int part = threadIdx.x / 32;
  float s = 0.0f;
  if (col < columns)
    for (int64_t r = part; r < shares; r += 8) s += in[r * columns + col];
  __shared__ float sums[8][33];
  sums[part][threadIdx.x % 32] = s;
  __syncthreads();
  if (part == 0 && col < columns) {
    for (int q = 1; q < 8; ++q) s += sums[q][threadIdx.x];
    const int64_t n = col / channels, d = col - n * channels;
    if (n < states) {
      if (dA) dA[d * states + n] = s;
    } else if (n == states) {
      if (dD) dD[d] = s;
    } else if (dbias) {
      dbias[d] = s;
    }
  }
}

// ---- single rows -------------------------------------------------------------------------------------------------------------------
// Bound by the states it reads and writes (8 bytes per channel and state).  A lane has 4 states of a channel (16 bytes: a wave's lanes
// read 1 KB in a row), LPC lanes a channel; y's sum over the lanes of a channel goes through DPP / lane swaps.
template <int LPC> __device__ inline float sum_neighbours(float v) {
  if constexpr (LPC >= 2) v += dpp<DPP_SWAP_1>(v);
  if constexpr (LPC >= 4) v += dpp<DPP_SWAP_2>(v);
  if constexpr (LPC >= 8) v += dpp<DPP_MIRROR_8>(v);
  if constexpr (LPC >= 16) v += dpp<DPP_ROTATE_8>(v);
  return v;
}

template <typename T, int LPC, bool WIDE>
__global__ void __launch_bounds__(256) scan_step(ppn_scan_step_args a) {
  const int64_t row = blockIdx.x;
  const int state = row_state(a.env_ids, row, a.environments);
  const int part = threadIdx.x % LPC, n0 = part * 4;
  const int64_t wide = a.channels / a.groups;
  const int64_t env = a.env_ids && state == ROW_LIVE ? a.env_ids[row] : row;
  const bool begins = a.starts && a.starts[row];
  for (int64_t d0 = (int64_t)blockIdx.y * (256 / LPC); d0 < a.channels; d0 += (int64_t)gridDim.y * (256 / LPC)) {
    const int64_t d = d0 + threadIdx.x / LPC;
    const bool live = d < a.channels;
    T* y = (T*)a.y + row * a.y_row + d;
    if (state != ROW_LIVE) {
      if (live && part == 0) *y = (T)(state == ROW_PADDING ? 0.0f : __builtin_nanf(""));
      continue;
    }
    float s = 0.0f, xv = 0.0f, zv = 0.0f;
    if (live) {
      const int64_t g = d / wide;
      float* hp = a.state + (env * a.channels + d) * a.states + n0;
      const float* ap = a.A + d * a.states + n0;
      const T* bp = (const T*)a.B + row * a.B_row + g * a.B_group + n0;
      const T* cp = (const T*)a.C + row * a.C_row + g * a.C_group + n0;
      float h[4], A2[4], bv[4], cv[4];
      if constexpr (WIDE) {
        const bool in = n0 < a.states;
        float4 h4 = in ? *(const float4*)hp : float4{0, 0, 0, 0}, a4 = in ? *(const float4*)ap : float4{0, 0, 0, 0};
        h[0] = h4.x, h[1] = h4.y, h[2] = h4.z, h[3] = h4.w;
        A2[0] = a4.x, A2[1] = a4.y, A2[2] = a4.z, A2[3] = a4.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = n0 + i < a.states;
        if constexpr (!WIDE) h[i] = in ? hp[i] : 0.0f, A2[i] = in ? ap[i] : 0.0f;
        bv[i] = in ? to_float(bp[i]) : 0.0f;
        cv[i] = in ? to_float(cp[i]) : 0.0f;
      }
      xv = to_float(((const T*)a.x)[row * a.x_row + d]);
      const float delta = step_size(to_float(((const T*)a.dt)[row * a.dt_row + d]), a.dt_bias ? a.dt_bias[d] : 0.0f, a.softplus);
      if (a.z) zv = to_float(((const T*)a.z)[row * a.z_row + d]);
      const float w = delta * xv;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[i] = begins ? w * bv[i] : __builtin_amdgcn_exp2f(delta * A2[i] * LOG2E) * h[i] + w * bv[i];
        s += cv[i] * h[i];
      }
      if constexpr (WIDE) {
        if (n0 < a.states) *(float4*)hp = float4{h[0], h[1], h[2], h[3]};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n0 + i < a.states) hp[i] = h[i];
      }
    }
    s = sum_neighbours<LPC>(s);
    if (live && part == 0) {
      if (a.D) s += a.D[d] * xv;
      if (a.z) s *= zv * sigmoid(zv);
      *y = (T)s;
    }
  }
}

// ---- plans -------------------------------------------------------------------------------------------------------------------------
template <typename F> int by_states(int64_t states, F f) {
  if (states <= 8) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
  if (states <= 16) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
  if (states <= 32) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 2>());
  return f(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
}

int64_t tiles_of(const ppn_scan_args* a) {
  const int64_t channels = a->states <= 16 ? 64 : a->states <= 32 ? 32 : 16;
  return ceil_div(a->channels / a->groups, channels);
}

// Chunks of time that are worked on at once: one while the waves of (environment, tile) alone fill the chip, since splitting walks the rows
// twice; else as many as bring `wanted` waves, of at least 32 rows.
struct Split { int64_t chunk, chunks; };
Split split_time(const ppn_scan_args* a, int64_t waves, int64_t wanted) {
  int64_t chunks = waves * 2 > wanted ? 1 : ceil_div(wanted, waves < 1 ? 1 : waves);
  int64_t chunk = ceil_div(ceil_div(a->time, chunks), ROWS) * ROWS;
  if (chunk < 32) chunk = 32;
  if (ceil_div(a->time, chunk) > 65535) chunk = ceil_div(ceil_div(a->time, 65535), ROWS) * ROWS;
  chunks = a->time ? ceil_div(a->time, chunk) : 1;
  return {chunk, chunks < 1 ? 1 : chunks};
}
Split forward_split(const ppn_scan_args* a) { return split_time(a, a->batch * a->groups * tiles_of(a), 4096); }

struct BackwardPlan { Split split; int64_t share, shares, rows_bytes, params_bytes, ends_bytes, sums_bytes; };
BackwardPlan plan_backward(const ppn_scan_args* a) {
  BackwardPlan p;
  const int64_t tiles = a->groups * tiles_of(a);
  p.split = split_time(a, a->batch * tiles, 2048);
  // environments per wave: one row of partial parameter gradients each, so as few as keep 2048 waves (two for each SIMD)
  p.share = p.split.chunks > 1 ? 1 : a->batch * tiles / 2048;
  if (p.share < 1) p.share = 1;
  p.shares = ceil_div(a->batch, p.share);
  auto round = [](int64_t v) { return (v + 255) / 256 * 256; };
  p.rows_bytes = round(tiles_of(a) * a->batch * a->time * a->groups * 2 * a->states * 4);
  p.params_bytes = round(p.shares * p.split.chunks * (a->states + 2) * a->channels * 4);
  p.ends_bytes = p.split.chunks > 1 ? round(a->batch * p.split.chunks * a->states * a->channels * 4) : 0;
  p.sums_bytes = p.split.chunks > 1 ? round(a->batch * p.split.chunks * 2 * a->channels * 4) : 0;
  return p;
}

int check(const ppn_scan_args* a) {
  if (!a || a->struct_bytes != (int64_t)sizeof *a) return fail(PPN_E_INVALID, "ppn_scan_args: struct_bytes does not match this library");
  if (a->type < 0 || a->type > PPN_T_F16) return fail(PPN_E_INVALID, "element type %lld is unknown", (long long)a->type);
  if (a->batch < 0 || a->time < 0 || a->channels < 1 || a->groups < 1 || a->channels % a->groups)
    return fail(PPN_E_INVALID, "scan: batch, time >= 0 and channels a multiple of groups >= 1 are needed");
  if (a->batch > 0x7fffffff || a->time > 0x7fffffff || a->channels > (1 << 24)) return fail(PPN_E_INVALID, "scan: a size is out of range");
  if (a->states < 1 || a->states > 64) return fail(PPN_E_INVALID, "states must be 1..64, got %lld", (long long)a->states);
  return PPN_OK;
}

}  // namespace
}  // namespace ppn_policy

using namespace ppn_policy;

extern "C" int64_t ppn_scan_checkpoint_bytes(const ppn_scan_args* a) {
  if (int rc = check(a)) return rc;
  return a->batch * ceil_div(a->time, ROWS) * a->states * a->channels * 4;
}

extern "C" int64_t ppn_scan_forward_workspace(const ppn_scan_args* a) {
  if (int rc = check(a)) return rc;
  const Split s = forward_split(a);
  return s.chunks > 1 ? a->batch * s.chunks * (a->states + 2) * a->channels * 4 : 0;
}

extern "C" int ppn_scan_forward(const ppn_scan_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  if (a->batch == 0) return PPN_OK;
  if (!a->A || (a->time && (!a->x || !a->dt || !a->B || !a->C || !a->y))) return fail(PPN_E_INVALID, "ppn_scan_forward: x, dt, A, B, C and y are needed");
  const Split s = forward_split(a);
  if (a->workspace_bytes < ppn_scan_forward_workspace(a) || (s.chunks > 1 && !a->workspace)) return fail(PPN_E_INVALID, "ppn_scan_forward: the workspace is too small");
  const int64_t waves = a->batch * a->groups * tiles_of(a), cells = a->batch * a->states * a->channels;
  if (waves > 0x7fffffff || ceil_div(cells, 256) > 0x7fffffff) return fail(PPN_E_INVALID, "scan: too many channels of too many environments");
  const dim3 grid(waves, s.chunks);
  float* ends = (float*)a->workspace;
  float* sums = ends + cells * s.chunks;
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return by_states(a->states, [&](auto ns, auto lpc) {
      constexpr int NS = decltype(ns)::value, LPC = decltype(lpc)::value;
      if (s.chunks > 1) {
        scan_forward<T, NS, LPC, true><<<grid, dim3(64), 0, (hipStream_t)stream>>>(*a, s.chunk, s.chunks, nullptr, ends, sums);
        scan_join<false><<<dim3(ceil_div(cells, 256)), dim3(256), 0, (hipStream_t)stream>>>(*a, s.chunks, ends, sums);
      }
      scan_forward<T, NS, LPC, false><<<grid, dim3(64), 0, (hipStream_t)stream>>>(*a, s.chunk, s.chunks, s.chunks > 1 ? ends : nullptr, nullptr, nullptr);
      return launched("ppn_scan_forward");
    });
  });
}

extern "C" int64_t ppn_scan_backward_workspace(const ppn_scan_args* a) {
  if (int rc = check(a)) return rc;
  const BackwardPlan p = plan_backward(a);
  return p.rows_bytes + p.params_bytes + p.ends_bytes + p.sums_bytes;
}

extern "C" int ppn_scan_backward(const ppn_scan_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  if (a->batch == 0 || a->time == 0) return fail(PPN_E_INVALID, "ppn_scan_backward: there are no rows");
  if (!a->x || !a->dt || !a->A || !a->B || !a->C || !a->dy || !a->dx || !a->ddt || !a->dB || !a->dC || !a->checkpoints)
    return fail(PPN_E_INVALID, "ppn_scan_backward: x, dt, A, B, C, dy, dx, ddt, dB, dC and checkpoints are needed");
  if (!a->z != !a->dz && a->dz) return fail(PPN_E_INVALID, "ppn_scan_backward: dz without z");
  const BackwardPlan p = plan_backward(a);
  if (!a->workspace || a->workspace_bytes < ppn_scan_backward_workspace(a)) return fail(PPN_E_INVALID, "ppn_scan_backward: the workspace is too small");
  char* w = (char*)a->workspace;
  float* rows = (float*)w;
  float* params = (float*)(w + p.rows_bytes);
  float* ends = (float*)(w + p.rows_bytes + p.params_bytes);
  float* sums = (float*)(w + p.rows_bytes + p.params_bytes + p.ends_bytes);
  const int64_t tiles = a->groups * tiles_of(a), cells = a->batch * a->states * a->channels, count = a->batch * a->time * a->groups * 2 * a->states;
  if (p.shares * tiles > 0x7fffffff || ceil_div(cells, 256) > 0x7fffffff || ceil_div(count, 256) > 0x7fffffff) return fail(PPN_E_INVALID, "scan: too many rows");
  const dim3 grid(p.shares * tiles, p.split.chunks);
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return by_states(a->states, [&](auto ns, auto lpc) {
      constexpr int NS = decltype(ns)::value, LPC = decltype(lpc)::value;
      const bool split = p.split.chunks > 1;
      if (split) {
        scan_backward<T, NS, LPC, true><<<grid, dim3(64), 0, (hipStream_t)stream>>>(*a, p.split.chunk, p.split.chunks, p.share, nullptr, ends, sums, nullptr, nullptr);
        scan_join<true><<<dim3(ceil_div(cells, 256)), dim3(256), 0, (hipStream_t)stream>>>(*a, p.split.chunks, ends, sums);
      }
      scan_backward<T, NS, LPC, false><<<grid, dim3(64), 0, (hipStream_t)stream>>>(*a, p.split.chunk, p.split.chunks, p.share, split ? ends : nullptr, nullptr, nullptr, rows, params);
      scan_reduce_rows<T><<<dim3(ceil_div(count, 256)), dim3(256), 0, (hipStream_t)stream>>>(rows, tiles_of(a), a->batch * a->time * a->groups, a->states, (T*)a->dB, (T*)a->dC);
      scan_reduce_params<<<dim3(ceil_div((a->states + 2) * a->channels, 32)), dim3(256), 0, (hipStream_t)stream>>>(params, p.shares * p.split.chunks, a->states,
                                                                                                                   a->channels, a->dA, a->dD, a->ddt_bias);
      return launched("ppn_scan_backward");
    });
  });
}

extern "C" int ppn_scan_step(const ppn_scan_step_args* a, void* stream) {
  if (!a || a->struct_bytes != (int64_t)sizeof *a) return fail(PPN_E_INVALID, "ppn_scan_step_args: struct_bytes does not match this library");
  if (a->rows < 0 || a->environments < 0 || a->channels < 1 || a->channels > (1 << 24) || a->rows > 0x7fffffff || a->groups < 1 || a->channels % a->groups)
    return fail(PPN_E_INVALID, "ppn_scan_step: a size is out of range");
  if (a->states < 1 || a->states > 64) return fail(PPN_E_INVALID, "states must be 1..64, got %lld", (long long)a->states);
  if (!a->env_ids && a->rows > a->environments) return fail(PPN_E_INVALID, "ppn_scan_step: more rows than environments and no env_ids");
  if (a->rows == 0) return PPN_OK;
  if (!a->x || !a->dt || !a->A || !a->B || !a->C || !a->y || (!a->state && a->environments)) return fail(PPN_E_INVALID, "ppn_scan_step: x, dt, A, B, C, state and y are needed");
  const bool wide = a->states % 4 == 0 && aligned(a->state, 16) && aligned(a->A, 16);
  int lpc = 1;
  while (lpc * 4 < a->states) lpc *= 2;
  // a workgroup takes all channels of its row (the ids in front of it are compared once) unless there are too few rows to fill the chip
  const int64_t slices = ceil_div(a->channels, 256 / lpc);
  int64_t y = ceil_div(1024, a->rows);
  if (y > slices) y = slices;
  if (y > 65535) y = 65535;
  const dim3 grid(a->rows, y);
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    auto go = [&](auto l) {
      constexpr int LPC = decltype(l)::value;
      if (wide) scan_step<T, LPC, true><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a);
      else scan_step<T, LPC, false><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a);
      return launched("ppn_scan_step");
    };
    switch (lpc) {
      case 1: return go(std::integral_constant<int, 1>());
      case 2: return go(std::integral_constant<int, 2>());
      case 4: return go(std::integral_constant<int, 4>());
      case 8: return go(std::integral_constant<int, 8>());
    }
    return go(std::integral_constant<int, 16>());
  });
}
