// ppn_scan.hip -- the selective state space scan of a policy's memory: whole windows, their gradients, single rows.
//
//   h[t,d,n] = exp(delta A[d,n]) h[t-1,d,n] + delta B[t,n] x[t,d]      delta = softplus(dt + dt_bias)
//   y[t,d]   = (sum_n C[t,n] h[t,d,n] + D[d] x[t,d]) silu(z[t,d])
//
// Bound by the vector units: every element (environment, row, channel) takes one exponential (2.7 slots of 4 clocks a wave, counted) and four
// multiplications and additions per state, against 4 elements moved: 8 instructions a state forward, 27 backward, with all that is done once a
// row.  Hence: one lane owns one channel with all its states in registers (two or four lanes above 16 and 32 states), nothing is
// exchanged between lanes in the forward pass, and B and C (the same for all lanes of a wave) are read once per wave and 8 rows, widened
// to 32 bits in LDS and broadcast from there.  Workgroups are single waves: no barrier is waited for.
//
// A window of 1024 x 60 rows of 512 bfloat16 channels with 16 states, for training, behind a hundred others (the card's clock rises over the first tens):
// forward 178 us (vector units 68 % busy; 520 MB, half of them checkpoints), backward 485 us (87 %), the sums 27 us.  Twice 8724 rows of 768 float16
// channels, no gradients: 49 us for the chunks' ends, 18 us to join them, 62 us for y.  Fetching a block ahead, into registers or straight into LDS, made none of these faster.
#include "ppn_policy.h"

namespace ppn_policy {
namespace {

constexpr int ROWS = 8;          // rows of a block; also the distance of the checkpoints the backward pass restarts from

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
  __device__ static int first(int lane) { return ((lane & ((1 << LEVELS) - 1)) >> SPARE) * COUNT; }
};

// ---- staging -----------------------------------------------------------------------------------------------------------------------
// The rows are taken in blocks of ROWS without a branch that a memory operation hangs on: the wait for a block's loads would otherwise be a
// wait for every store before them too.  A block past the end of the time axis (or of the chunk) repeats its last row, which leaves the state as it
// is and writes the last row's values again; a lane past the last channel, and the second and
// later lanes of a channel, write what the channel's own lane writes.

// Addresses are a pointer that is the same for the wave, in scalar registers, and an unsigned 32-bit byte offset.  A block's rows lie within such
// an offset: strides of time are at most 2^27 elements, as the entry points check.
template <typename V> __device__ inline V& at(const void* base, unsigned bytes) { return *(V*)((char*)base + bytes); }

// Loads waited for here: else the first round's waits, which have few operations behind them, stand in every round of the loop that follows.
template <typename V> __device__ inline void settled(V& v) { asm volatile("" : "+v"(v)); }

// ROWS rows of B and C of one environment and group, as 32-bit floats in LDS, zero beyond the last state: fetched into registers with the block's
// other loads, put into LDS when all are in.
template <typename T, int STATES, bool WITH_B, bool WITH_C> struct Staged {
  static constexpr int COUNT = ROWS * STATES / 64;
  T b[COUNT], c[COUNT];
  __device__ void fetch(const ppn_scan_args& a, const T* B, const T* C, int rows) {      // B, C: at the block's first row
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const int e = threadIdx.x + 64 * i, j = min(e / STATES, rows - 1), n = min(e % STATES, (int)a.states - 1);
      if constexpr (WITH_B) b[i] = at<const T>(B, ((unsigned)j * (unsigned)a.B_time + (unsigned)n) * (unsigned)sizeof(T));
      if constexpr (WITH_C) c[i] = at<const T>(C, ((unsigned)j * (unsigned)a.C_time + (unsigned)n) * (unsigned)sizeof(T));
    }
  }
  __device__ void put(int states, float* sb, float* sc) const {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const int e = threadIdx.x + 64 * i;
      if constexpr (WITH_B) sb[e] = e % STATES < states ? to_float(b[i]) : 0.0f;
      if constexpr (WITH_C) sc[e] = e % STATES < states ? to_float(c[i]) : 0.0f;
    }
  }
};

template <int NS> __device__ inline void read_states(const float* p, float (&v)[NS]) {
#pragma unroll
  for (int i = 0; i < NS; i += 4) {
    float4 q = *(const float4*)(p + i);
    v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
  }
}

// One block's rows of a [.. x channels] tensor, this lane's channel: ROWS loads in flight.
template <typename T> struct Column {
  T v[ROWS];
  __device__ void fetch(const T* p, int64_t stride, unsigned d, int rows) {
    const unsigned step = (unsigned)stride * (unsigned)sizeof(T);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) v[j] = at<const T>(p, (unsigned)min(j, rows - 1) * step + d * (unsigned)sizeof(T));
  }
};

// A value the compiler knows nothing about: what follows is computed from it here, not moved in front of earlier rows or kept from them (eight rows'
// exponentials, B and C do not fit the registers next to the states).
__device__ inline float anew(float v) {
  asm volatile("" : "+v"(v)::"memory");
  __builtin_amdgcn_sched_barrier(0);
  return v;
}
template <typename T> __device__ inline float widened(T v) {      // to_float, here and not in front of earlier rows
  float f = to_float(v);
  asm volatile("" : "+v"(f));
  return f;
}

// Bit j: row t0 + j begins an episode.  Wave-uniform.
__device__ inline unsigned starts_of(const ppn_scan_args& a, int64_t b, int64_t t0, int rows) {
  if (!a.starts) return 0;
  const int lane = threadIdx.x, j = min(lane, rows - 1);
  const bool s = a.starts[b * a.starts_batch + (t0 + j) * a.starts_time] != 0;
  return (unsigned)__ballot(s && lane < rows);
}

// d: this lane's channel, as an unsigned offset from a row's address, which is the same for the wave and kept in scalar registers.
struct Place { int64_t b, g, tile; unsigned d; bool live; int part; };

// Workgroup x: (environment, group, tile of channels), the tile fastest.  The eight dies take workgroups in turn, each with its own L2: neighbours
// in that order (which share rows of B and C, and cache lines where a tile's rows end inside one) are given to one die.  A lane past the last
// channel works on the last one.
template <int NS, int LPC> __device__ inline Place place(const ppn_scan_args& a) {
  constexpr unsigned CHANNELS = Shape<NS, LPC>::CHANNELS;
  const unsigned per = gridDim.x / 8, x = blockIdx.x < per * 8 ? (blockIdx.x % 8) * per + blockIdx.x / 8 : blockIdx.x;
  const unsigned groups = (unsigned)a.groups, wide = (unsigned)a.channels / groups, tiles = (wide + CHANNELS - 1) / CHANNELS;
  const unsigned b = x / (groups * tiles), gt = x - b * (groups * tiles), g = gt / tiles, tile = gt - g * tiles;
  Place p;
  p.b = __builtin_amdgcn_readfirstlane((int)b);
  p.g = __builtin_amdgcn_readfirstlane((int)g);
  p.tile = __builtin_amdgcn_readfirstlane((int)tile);
  const unsigned c = tile * CHANNELS + threadIdx.x % CHANNELS;
  p.live = c < wide;
  p.d = g * wide + (p.live ? c : wide - 1);
  p.part = threadIdx.x / CHANNELS;
  return p;
}

// Row-major [.. x channels x states] tensors of the caller (A, initial and final states).
template <int NS> __device__ inline void load_states(const float* p, int64_t states, int part, float (&v)[NS]) {
#pragma unroll
  for (int n = 0; n < NS; ++n) v[n] = p[min(part * NS + n, (int)states - 1)];      // (a branch for the last ones would wait for each load in turn)
#pragma unroll
  for (int n = 0; n < NS; ++n) v[n] = part * NS + n < (int)states ? v[n] : 0.0f;
}
template <int NS> __device__ inline void store_states(float* p, int64_t states, int part, const float (&v)[NS]) {
#pragma unroll
  for (int n = 0; n < NS; ++n)
    if (part * NS + n < states) p[part * NS + n] = v[n];
}
// Workspace states: [.. x states x channels], so that a wave's lanes write next to each other.  Places past the last state are read as the last one
// (and do not matter: B and C are zero there).
template <int NS, int LPC> __device__ inline void load_plane(const float* p, int64_t states, int64_t channels, unsigned d, int part, float (&v)[NS]) {
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    if constexpr (LPC == 1) v[n] = at<const float>(p + min(n, (int)states - 1) * channels, d * 4u);
    else v[n] = at<const float>(p, ((unsigned)min(part * NS + n, (int)states - 1) * (unsigned)channels + d) * 4u);
  }
}
template <int NS, int LPC> __device__ inline void store_plane(float* p, int64_t states, int64_t channels, unsigned d, int part, const float (&v)[NS]) {
#pragma unroll
  for (int n = 0; n < NS; ++n)
    if (part * NS + n < (int)states) {
      if constexpr (LPC == 1) at<float>(p + n * channels, d * 4u) = v[n];
      else at<float>(p, ((unsigned)(part * NS + n) * (unsigned)channels + d) * 4u) = v[n];
    }
}

// softplus of a block's step sizes at once (one branch); rows past the block's last one: 0.
template <typename T> __device__ inline void step_sizes(const Column<T>& dt, float bias, bool soft, int rows, float (&delta)[ROWS]) {
#pragma unroll
  for (int j = 0; j < ROWS; ++j) delta[j] = to_float(dt.v[j]) + bias;
  if (soft) {
#pragma unroll
    for (int j = 0; j < ROWS; ++j) delta[j] = softplus(delta[j]);
  }
#pragma unroll
  for (int j = 1; j < ROWS; ++j) delta[j] = j < rows ? delta[j] : 0.0f;
}

// The state behind a row; a row that begins an episode drops the state before, whatever is in it, and a repeated row (past the block's last one) leaves it,
// whatever the row holds: a step size of zero times an infinity would not (branches the whole wave takes).
template <int NS> __device__ inline void advance(const float (&before)[NS], float (&h)[NS], float delta, float w, const float (&A2)[NS], const float (&bv)[NS], bool begin, bool real) {
  if (begin) {
#pragma unroll
    for (int n = 0; n < NS; ++n) h[n] = w * bv[n];
  } else if (real) {
#pragma unroll
    for (int n = 0; n < NS; ++n) h[n] = __builtin_amdgcn_exp2f(delta * A2[n]) * before[n] + w * bv[n];
  } else {
#pragma unroll
    for (int n = 0; n < NS; ++n) h[n] = before[n];
  }
}

// What a chunk leaves of a state that enters it: exp2(rate) h, where the exponential may pass 32 bits and the product need not (A > 0 or delta < 0; a state
// of zero stays zero).  In two halves: what 2^256 does to a number is beyond 32 bits anyway.
__device__ inline float carried(float rate, float h) {
  const float half = __builtin_amdgcn_exp2f(0.5f * rate);
  return h == 0.0f ? h : half * (half * h);
}

// What enters a chunk, from what the chunks before it do (`count` of them, from `first` in steps of `step`), in h: as scan_join, in the wave that goes on
// with it.
template <int NS, int LPC>
__device__ inline void join_chunks(const ppn_scan_args& a, const Place& p, int64_t chunks, const float* ends, const float* sums, int first, int count, int step,
                                   const float (&A2)[NS], float (&h)[NS]) {
  constexpr int AHEAD = 2;
  const int64_t plane = a.states * a.channels;
  for (int i0 = 0; i0 < count; i0 += AHEAD) {
    float own[AHEAD][NS], total[AHEAD], cut[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int64_t at_chunk = p.b * chunks + first + step * min(i0 + j, count - 1);
      load_plane<NS, LPC>(ends + at_chunk * plane, a.states, a.channels, p.d, p.part, own[j]);
      total[j] = at<const float>(sums + (at_chunk * 2 + 0) * a.channels, p.d * 4u);
      cut[j] = at<const float>(sums + (at_chunk * 2 + 1) * a.channels, p.d * 4u);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i0 + j < count) {
#pragma unroll
        for (int n = 0; n < NS; ++n) h[n] = cut[j] != 0.0f ? own[j][n] : own[j][n] + carried(total[j] * A2[n], h[n]);
      }
  }
}

// ---- forward -----------------------------------------------------------------------------------------------------------------------
// One wave: 64 / LPC channels of one environment over the rows of one chunk (grid.y chunks of `chunk` rows, a multiple of ROWS).
// OUTPUT: y.  TRAIN: the states in front of every block as well.  SUMMARY: neither, only what the chunk does to a state that enters it: its
// own end state from zero, the sum of delta (the decay of the whole chunk is exp(A sum delta)), and whether an episode's start cuts it.
enum { OUTPUT, TRAIN, SUMMARY };
template <typename T, int NS, int LPC, int MODE>
__global__ void __launch_bounds__(64, 4) scan_forward(ppn_scan_args a, int64_t chunk, int64_t chunks, const float* entering, float* ends, float* sums) {
  constexpr int STATES = Shape<NS, LPC>::STATES;
  __shared__ __align__(16) float sb[ROWS * STATES], sc[ROWS * STATES];
  const Place p = place<NS, LPC>(a);
  const int64_t k = blockIdx.y, t0 = k * chunk, t1 = t0 + chunk < a.time ? t0 + chunk : a.time, plane = a.states * a.channels;
  float A2[NS], h[NS];
  load_states<NS>(a.A + (int64_t)p.d * a.states, a.states, p.part, A2);
#pragma unroll
  for (int n = 0; n < NS; ++n) A2[n] *= LOG2E, h[n] = 0.0f;
  if constexpr (MODE != SUMMARY) {
    if (entering) load_plane<NS, LPC>(entering + (p.b * chunks + k) * plane, a.states, a.channels, p.d, p.part, h);
    else if (a.initial) load_states<NS>(a.initial + (p.b * a.channels + p.d) * a.states, a.states, p.part, h);
    if (ends) join_chunks<NS, LPC>(a, p, chunks, ends, sums, 0, (int)k, 1, A2, h);
  }
  const float bias = a.dt_bias ? a.dt_bias[p.d] : 0.0f, skip = a.D ? a.D[p.d] : 0.0f;
  const bool soft = a.softplus, gated = a.z != nullptr;
  // (without a gate, x is read in its place)
  const void* zz = gated ? a.z : a.x;
  const int64_t z_batch = gated ? a.z_batch : a.x_batch, z_time = gated ? a.z_time : a.x_time;
  const T* px = (const T*)a.x + p.b * a.x_batch + t0 * a.x_time;
  const T* pdt = (const T*)a.dt + p.b * a.dt_batch + t0 * a.dt_time;
  const T* pz = (const T*)zz + p.b * z_batch + t0 * z_time;
  const T* pB = (const T*)a.B + p.b * a.B_batch + p.g * a.B_group + t0 * a.B_time;
  const T* pC = (const T*)a.C + p.b * a.C_batch + p.g * a.C_group + t0 * a.C_time;
  T* py = (T*)a.y + p.b * a.y_batch + t0 * a.y_time;
  float* pmark = MODE == TRAIN ? a.checkpoints + (p.b * ((a.time + ROWS - 1) / ROWS) + t0 / ROWS) * plane : nullptr;
  const unsigned y_step = (unsigned)a.y_time;
  float total = 0.0f;
  bool cut = false;
#pragma unroll
  for (int n = 0; n < NS; ++n) settled(A2[n]), settled(h[n]);
  for (int64_t t = t0; t < t1; t += ROWS) {
    const int rows = (int)min(t1 - t, (int64_t)ROWS);
    Column<T> x, dt, z;
    Staged<T, STATES, true, MODE != SUMMARY> bc;
    dt.fetch(pdt, a.dt_time, p.d, rows);
    x.fetch(px, a.x_time, p.d, rows);
    bc.fetch(a, pB, pC, rows);
    if constexpr (MODE != SUMMARY) z.fetch(pz, z_time, p.d, rows);
    const unsigned now = starts_of(a, p.b, t, rows);
    px += ROWS * a.x_time, pdt += ROWS * a.dt_time, pz += ROWS * z_time, pB += ROWS * a.B_time, pC += ROWS * a.C_time;
    cut |= now != 0;
    float delta[ROWS], gate[ROWS];
    step_sizes(dt, bias, soft, rows, delta);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      if constexpr (MODE == SUMMARY) {
        total += delta[j];
      } else {
        const float zv = to_float(z.v[j]);
        gate[j] = gated ? zv * sigmoid(zv) : 1.0f;
      }
    }
    __syncthreads();
    bc.put((int)a.states, sb, sc);
    __syncthreads();
    if constexpr (MODE == TRAIN) {
      store_plane<NS, LPC>(pmark, a.states, a.channels, p.d, p.part, h);
      pmark += plane;
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      float bv[NS];
      const float step = anew(delta[j]);
      read_states<NS>(sb + j * STATES + p.part * NS, bv);
      const float xv = widened(x.v[j]);
      advance<NS>(h, h, step, step * xv, A2, bv, (now >> j) & 1, j < rows);
      if constexpr (MODE != SUMMARY) {
        float cv[NS], s = 0.0f;
        read_states<NS>(sc + j * STATES + p.part * NS, cv);
#pragma unroll
        for (int n = 0; n < NS; ++n) s += cv[n] * h[n];
        at<T>(py + (uint64_t)((unsigned)min(j, rows - 1) * y_step), p.d * (unsigned)sizeof(T)) = (T)((sum_parts<LPC>(s) + skip * xv) * gate[j]);
      }
    }
    py += ROWS * a.y_time;
  }
  if constexpr (MODE == SUMMARY) {
    store_plane<NS, LPC>(ends + (p.b * chunks + k) * plane, a.states, a.channels, p.d, p.part, h);
    sums[((p.b * chunks + k) * 2 + 0) * a.channels + p.d] = total;
    sums[((p.b * chunks + k) * 2 + 1) * a.channels + p.d] = cut ? 1.0f : 0.0f;
  } else if (a.final_state && t1 == a.time) {
    store_states<NS>(a.final_state + (p.b * a.channels + p.d) * a.states, a.states, p.part, h);
  }
}

// What enters each chunk, in place of what leaves it (forward: chunk k from k - 1; BACKWARD: adjoints, chunk k from k + 1).
template <bool BACKWARD>
__global__ void __launch_bounds__(64) scan_join(ppn_scan_args a, int64_t chunks, float* ends, const float* sums) {
  const int64_t id = (int64_t)blockIdx.x * 64 + threadIdx.x, per = a.states * a.channels;
  if (id >= a.batch * per) return;
  const int64_t b = id / per, rest = id - b * per, n = rest / a.channels, d = rest - n * a.channels;
  const float A2 = a.A[d * a.states + n] * LOG2E;
  const float* outside = BACKWARD ? a.dfinal : a.initial;
  float h = outside ? outside[(b * a.channels + d) * a.states + n] : 0.0f;
  float* p = ends + b * chunks * per + rest;
  const float* s = sums + b * chunks * 2 * a.channels + d;
  constexpr int AHEAD = 16;
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
      h = cut[j] != 0.0f ? own[j] : own[j] + carried(total[j] * A2, h);
    }
  }
}

// ---- backward ----------------------------------------------------------------------------------------------------------------------
// With u[t] = dy[t] silu(z[t]) and the adjoint e[t] = u[t] C[t] + exp(delta[t+1] A) e[t+1]  (0 across an episode's start):
//   dC[t] = sum_d u[t] h[t]       dB[t] = sum_d e[t] delta[t] x[t]       dx[t] = delta[t] sum_n e[t] B[t] + D u[t]
//   q[t] = e[t] exp(delta[t] A) h[t-1];   ddelta[t] = sum_n q[t] A + x[t] sum_n e[t] B[t];   dA = sum_t q[t] delta[t]
// The rows are taken in blocks of 8 from the last to the first.  A block's states are recomputed from its checkpoint, four rows' worth kept in
// registers at a time with 16 states a lane (5 x 16; the first four rows are walked twice for that: 8 % more work, and two waves fit a SIMD
// where all eight rows' states left room for one), eight with 8 states.  The sums over channels (dB, dC) are the wave's part of them, one row of
// partial sums per tile of channels, added up by scan_reduce; dA, dD and ddt_bias stay in registers over the wave's rows and leave one
// row of partial sums for each environment and chunk.  Both reductions run in a fixed order.
//
// ENDS: only what a chunk adds to the adjoint in front of it, and its sum of delta, for chunks that are worked on at once.  JOINING: gradients, behind
// join_chunks (a kernel of its own: its registers cost the others 26 us of 690 in a training step).
enum { GRADIENTS, JOINING, ENDS };
template <typename T, int NS, int LPC, int MODE>
__global__ void __launch_bounds__(64, 2) scan_backward(ppn_scan_args a, int64_t chunk, int64_t chunks, const float* entering, float* ends, float* sums, float* rows_out,
                                                                    float* params_out) {
  constexpr bool ADJOINT = MODE == ENDS;
  constexpr int STATES = Shape<NS, LPC>::STATES, KEPT = NS == 8 ? ROWS : ROWS / 2;
  __shared__ __align__(16) float sb[ADJOINT ? 4 : ROWS * STATES], sc[ROWS * STATES];
  const Place p = place<NS, LPC>(a);
  const int64_t k = blockIdx.y, first = k * chunk, last = first + chunk < a.time ? first + chunk : a.time;
  const int64_t plane = a.states * a.channels, pair = a.groups * 2 * STATES, cell = p.b * chunks + k;
  const bool soft = a.softplus, gated = a.z != nullptr;
  const float alive = p.live ? 1.0f : 0.0f;
  int64_t t = (last - 1) / ROWS * ROWS;
  // without a gate: x in z's place, and dz goes where dx is written over it
  const bool dgate = a.dz != nullptr;
  const int64_t x_time = a.x_time, dt_time = a.dt_time, dy_time = a.dy_time, dx_time = a.dx_time, ddt_time = a.ddt_time;
  const int64_t z_time = gated ? a.z_time : x_time, dz_time = dgate ? a.dz_time : dx_time;
  const T* px = (const T*)a.x + p.b * a.x_batch + t * x_time;
  const T* pdt = (const T*)a.dt + p.b * a.dt_batch + t * dt_time;
  const T* pdy = (const T*)a.dy + p.b * a.dy_batch + t * dy_time;
  const T* pz = gated ? (const T*)a.z + p.b * a.z_batch + t * z_time : px;
  const T* pB = (const T*)a.B + p.b * a.B_batch + p.g * a.B_group + t * a.B_time;
  const T* pC = (const T*)a.C + p.b * a.C_batch + p.g * a.C_group + t * a.C_time;
  T* pdx = ADJOINT ? nullptr : (T*)a.dx + p.b * a.dx_batch + t * dx_time;
  T* pddt = ADJOINT ? nullptr : (T*)a.ddt + p.b * a.ddt_batch + t * ddt_time;
  T* pdz = ADJOINT ? nullptr : dgate ? (T*)a.dz + p.b * a.dz_batch + t * dz_time : pdx;
  const float* pmark = ADJOINT ? nullptr : a.checkpoints + (p.b * ((a.time + ROWS - 1) / ROWS) + t / ROWS) * plane;
  float* pout = ADJOINT ? nullptr : rows_out + ((p.tile * a.batch + p.b) * a.time + t) * pair + p.g * 2 * STATES;
  float A2[NS], dA[NS], e[NS];
  load_states<NS>(a.A + (int64_t)p.d * a.states, a.states, p.part, A2);
#pragma unroll
  for (int n = 0; n < NS; ++n) A2[n] *= LOG2E, dA[n] = 0.0f, e[n] = 0.0f;
  if constexpr (!ADJOINT) {
    if (entering) load_plane<NS, LPC>(entering + cell * plane, a.states, a.channels, p.d, p.part, e);
    else if (a.dfinal) load_states<NS>(a.dfinal + (p.b * a.channels + p.d) * a.states, a.states, p.part, e);
    if constexpr (MODE == JOINING) join_chunks<NS, LPC>(a, p, chunks, ends, sums, (int)chunks - 1, (int)(chunks - 1 - k), -1, A2, e);
  }
  const float bias = a.dt_bias ? a.dt_bias[p.d] : 0.0f, skip = a.D ? a.D[p.d] : 0.0f;
  const unsigned mine = p.d * (unsigned)sizeof(T);
  float dskip = 0.0f, dbias = 0.0f, total = 0.0f;
  bool cut = false;
#pragma unroll
  for (int n = 0; n < NS; ++n) settled(A2[n]), settled(e[n]);
  for (; t >= first; t -= ROWS) {
    const int rows = (int)min(last - t, (int64_t)ROWS);
    Column<T> x, dt, z, dy;
    Staged<T, STATES, !ADJOINT, true> bc;
    float mark[NS], h[ADJOINT ? 1 : KEPT + 1][NS], delta[ROWS];
    dt.fetch(pdt, dt_time, p.d, rows);
    bc.fetch(a, pB, pC, rows);
    if constexpr (!ADJOINT) load_plane<NS, LPC>(pmark, a.states, a.channels, p.d, p.part, mark);
    if constexpr (!ADJOINT) x.fetch(px, x_time, p.d, rows);
    dy.fetch(pdy, dy_time, p.d, rows);
    z.fetch(pz, z_time, p.d, rows);
    const unsigned now = starts_of(a, p.b, t, rows);
    px -= ROWS * x_time, pdt -= ROWS * dt_time, pdy -= ROWS * dy_time, pz -= ROWS * z_time, pB -= ROWS * a.B_time, pC -= ROWS * a.C_time;
    if constexpr (!ADJOINT) pmark -= plane;
    cut |= now != 0;
    step_sizes(dt, bias, soft, rows, delta);
    if constexpr (ADJOINT) {
#pragma unroll
      for (int j = 0; j < ROWS; ++j) total += delta[j];
    }
    __syncthreads();
    bc.put((int)a.states, sb, sc);
    __syncthreads();
    auto forward = [&](int j, const float (&before)[NS], float (&after)[NS]) {
      float bv[NS];
      const float step = anew(delta[j]);
      read_states<NS>(sb + j * STATES + p.part * NS, bv);
      advance<NS>(before, after, step, step * widened(x.v[j]), A2, bv, (now >> j) & 1, true);      // (what is behind the last row is not looked at)
    };
#pragma unroll
    for (int j = ROWS - 1; j >= 0; --j) {
      if constexpr (!ADJOINT) {
        if (j % KEPT == KEPT - 1) {          // the states in front of and behind rows j - KEPT + 1 .. j, from the checkpoint
#pragma unroll
          for (int n = 0; n < NS; ++n) h[0][n] = mark[n];
#pragma unroll
          for (int i = 0; i < j - KEPT + 1; ++i) forward(i, h[0], h[0]);
#pragma unroll
          for (int i = 0; i < KEPT; ++i) forward(j - KEPT + 1 + i, h[i], h[i + 1]);
        }
      }
      const bool begin = (now >> j) & 1;
      const float step = anew(delta[j]);
      unsigned place = (unsigned)min(j, rows - 1);
      asm volatile("" : "+s"(place));
      const float real = __builtin_bit_cast(float, (int)place == j ? 0x3f800000 : 0);      // (a repeated last row adds nothing, and is written over by itself)
      const float up = widened(dy.v[j]) * real, zv = widened(z.v[j]), sg = gated ? sigmoid(zv) : 1.0f, u = gated ? up * zv * sg : up;
      float cv[NS];
      read_states<NS>(sc + j * STATES + p.part * NS, cv);
      if constexpr (ADJOINT) {
        if (begin) {
#pragma unroll
          for (int n = 0; n < NS; ++n) e[n] = 0.0f;
        } else if (j < rows) {
#pragma unroll
          for (int n = 0; n < NS; ++n) e[n] = __builtin_amdgcn_exp2f(step * A2[n]) * (e[n] + u * cv[n]);
        }
      } else {
        float bv[NS], part[2 * NS], s = 0.0f, through = 0.0f, decay = 0.0f;
        read_states<NS>(sb + j * STATES + p.part * NS, bv);
        const float xv = widened(x.v[j]), ul = u * alive, wl = step * xv * alive;        // (a lane past the last channel adds nothing to the sums over channels)
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          s += cv[n] * h[j % KEPT + 1][n];
          e[n] += u * cv[n];
          part[NS + n] = ul * h[j % KEPT + 1][n];
          part[n] = wl * e[n];
          through += e[n] * bv[n];
        }
        if (begin) {
#pragma unroll
          for (int n = 0; n < NS; ++n) e[n] = 0.0f;
        } else if (j < rows) {
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            e[n] *= __builtin_amdgcn_exp2f(step * A2[n]);
            const float q = e[n] * h[j % KEPT][n];
            dA[n] += q * step;
            decay += q * A2[n];
          }
        }
        sum_channels<2 * NS, LPC>(part);
        typedef Kept<2 * NS, LPC> K;
#pragma unroll
        for (int i = 0; i < K::COUNT; ++i) {            // (lanes that hold copies write the same values)
          const int v = K::first(threadIdx.x) + i, n = p.part * NS + v % NS;
          at<float>(pout, (place * (unsigned)pair + (unsigned)((v / NS) * STATES + n)) * 4u) = part[i];
        }
        s = sum_parts<LPC>(s) + skip * xv;
        through = sum_parts<LPC>(through);
        decay = sum_parts<LPC>(decay) * (1.0f / LOG2E);
        const float v = widened(dt.v[j]) + bias;
        float dd = decay + through * xv;
        dd *= !soft || v > 20.0f ? 1.0f : sigmoid(v);
        dbias += dd * real;
        dskip += u * xv;
        at<T>(pdz, place * ((unsigned)dz_time * (unsigned)sizeof(T)) + mine) = (T)(up * s * sg * (1.0f + zv * (1.0f - sg)));
        at<T>(pdx, place * ((unsigned)dx_time * (unsigned)sizeof(T)) + mine) = (T)(through * step + skip * u);
        at<T>(pddt, place * ((unsigned)ddt_time * (unsigned)sizeof(T)) + mine) = (T)dd;
      }
    }
    if constexpr (!ADJOINT) pdx -= ROWS * dx_time, pddt -= ROWS * ddt_time, pdz -= ROWS * dz_time, pout -= ROWS * pair;
  }
  if constexpr (ADJOINT) {
    store_plane<NS, LPC>(ends + cell * plane, a.states, a.channels, p.d, p.part, e);
    sums[(cell * 2 + 0) * a.channels + p.d] = total;
    sums[(cell * 2 + 1) * a.channels + p.d] = cut ? 1.0f : 0.0f;
  } else {
    if (a.dinitial && first == 0) store_states<NS>(a.dinitial + (p.b * a.channels + p.d) * a.states, a.states, p.part, e);
    float* out = params_out + cell * (a.states + 2) * a.channels;
    store_plane<NS, LPC>(out, a.states, a.channels, p.d, p.part, dA);
    out[a.states * a.channels + p.d] = dskip;
    out[(a.states + 1) * a.channels + p.d] = dbias;
  }
}

// The backward pass's partial sums added up, in a fixed order: the first `row_blocks` workgroups make dB and dC out of the tiles' rows [tiles x rows
// x 2 STATES] (padded to the states of whole lanes; four states a lane), the others dA, dD and ddt_bias out of the waves' rows [shares x
// (states + 2) x channels] (32 columns a workgroup, 8 lanes a column).  One launch: 63 MB and 38 MB take 20 and 15 us one after the other.
struct ReduceArgs { const float* rows_in; int64_t tiles, rows; const float* params_in; int64_t shares, states, channels; void *dB, *dC; float *dA, *dD, *dbias; int64_t row_blocks; };
template <typename T, int STATES>
__global__ void __launch_bounds__(256) scan_reduce(ReduceArgs a) {
  if (blockIdx.x < a.row_blocks) {
    const int64_t id = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, count = a.rows * 2 * STATES, row = id / (2 * STATES);
    const int v = (int)(id % (2 * STATES)), n = v % STATES;
    if (id >= count || n >= a.states) return;
    float4 s = {0, 0, 0, 0};
    for (int64_t t = 0; t < a.tiles; ++t) {
      const float4 part = *(const float4*)(a.rows_in + t * count + id);
      s.x += part.x, s.y += part.y, s.z += part.z, s.w += part.w;
    }
    T* out = (T*)(v < STATES ? a.dB : a.dC) + row * a.states + n;
    const float sums[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.states) out[i] = (T)sums[i];
    return;
  }
  const int64_t columns = (a.states + 2) * a.channels, col = ((int64_t)blockIdx.x - a.row_blocks) * 32 + threadIdx.x % 32;
  const int part = threadIdx.x / 32;
  float s = 0.0f;
  if (col < columns)
    for (int64_t r = part; r < a.shares; r += 64) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = r + 8 * i < a.shares ? a.params_in[(r + 8 * i) * columns + col] : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
  __shared__ float sums[8][33];
  sums[part][threadIdx.x % 32] = s;
  __syncthreads();
  if (part == 0 && col < columns) {
    for (int q = 1; q < 8; ++q) s += sums[q][threadIdx.x];
    const int64_t n = col / a.channels, d = col - n * a.channels;
    if (n < a.states) {
      if (a.dA) a.dA[d * a.states + n] = s;
    } else if (n == a.states) {
      if (a.dD) a.dD[d] = s;
    } else if (a.dbias) {
      a.dbias[d] = s;
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

template <typename T> struct alignas(4 * sizeof(T)) Four { T v[4]; };

// WIDE: four states (and four of B and C) are one load.  AHEAD channels of a lane are loaded together, and the first of them before the ids
// are compared.
template <typename T, int LPC, bool WIDE, int AHEAD>
__global__ void __launch_bounds__(256) scan_step(ppn_scan_step_args a) {
  constexpr int PER = 256 / LPC;        // channels a workgroup takes at a time, AHEAD times over
  const int64_t row = blockIdx.x, env = row_env(a.env_ids, row, a.environments);
  const int part = threadIdx.x % LPC, n0 = part * 4, states = (int)a.states, channels = (int)a.channels, wide = (int)(a.channels / a.groups);
  const int last = min(n0, states - 1) & ~3;       // (a lane past the last state reads the last four)
  const bool begins = a.starts && a.starts[row], gated = a.z != nullptr, soft = a.softplus;
  const T* x = (const T*)a.x + row * a.x_row;
  const T* dt = (const T*)a.dt + row * a.dt_row;
  const T* z = gated ? (const T*)a.z + row * a.z_row : x;
  const T* B = (const T*)a.B + row * a.B_row;
  const T* C = (const T*)a.C + row * a.C_row;
  T* y = (T*)a.y + row * a.y_row;
  float* state = a.state + env * a.channels * a.states;
  Four<float> h[AHEAD], A[AHEAD];
  Four<T> b[AHEAD], c[AHEAD];
  T rx[AHEAD], rdt[AHEAD], rz[AHEAD];
  float bias[AHEAD], skip[AHEAD];
  auto fetch = [&](int d0) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int d = min(d0 + k * PER + (int)threadIdx.x / LPC, channels - 1), g = d / wide;
      if constexpr (WIDE) {
        h[k] = *(const Four<float>*)(state + (int64_t)d * states + last);
        A[k] = *(const Four<float>*)(a.A + (int64_t)d * states + last);
        b[k] = *(const Four<T>*)(B + g * a.B_group + last);
        c[k] = *(const Four<T>*)(C + g * a.C_group + last);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = min(n0 + i, states - 1);
          h[k].v[i] = state[(int64_t)d * states + n];
          A[k].v[i] = a.A[(int64_t)d * states + n];
          b[k].v[i] = B[g * a.B_group + n];
          c[k].v[i] = C[g * a.C_group + n];
        }
      }
      rx[k] = x[d];
      rdt[k] = dt[d];
      rz[k] = z[d];
      bias[k] = a.dt_bias ? a.dt_bias[d] : 0.0f;
      skip[k] = a.D ? a.D[d] : 0.0f;
    }
  };
  const int first = blockIdx.y * PER * AHEAD, step = gridDim.y * PER * AHEAD;
  fetch(first);
  const int live = row_state(a.env_ids, row, a.environments);
  for (int d0 = first; d0 < channels; d0 += step) {
    if (d0 != first) fetch(d0);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int d = d0 + k * PER + (int)threadIdx.x / LPC;
      const float xv = to_float(rx[k]), raw = to_float(rdt[k]) + bias[k], delta = soft ? softplus(raw) : raw, w = delta * xv;
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = n0 + i < states;
        const float bv = in ? to_float(b[k].v[i]) : 0.0f, cv = in ? to_float(c[k].v[i]) : 0.0f;
        h[k].v[i] = begins ? w * bv : __builtin_amdgcn_exp2f(delta * (A[k].v[i] * LOG2E)) * h[k].v[i] + w * bv;
        s += in ? cv * h[k].v[i] : 0.0f;
      }
      s = sum_neighbours<LPC>(s);
      if (live == ROW_LIVE && d < channels) {
        if constexpr (WIDE) {
          if (n0 < states) *(Four<float>*)(state + (int64_t)d * states + n0) = h[k];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n0 + i < states) state[(int64_t)d * states + n0 + i] = h[k].v[i];
        }
      }
      if (part == 0 && d < channels) {
        const float zv = to_float(rz[k]), gate = gated ? zv * sigmoid(zv) : 1.0f;
        y[d] = (T)(live == ROW_LIVE ? (s + skip[k] * xv) * gate : live == ROW_PADDING ? 0.0f : __builtin_nanf(""));
      }
    }
  }
}

// ---- plans -------------------------------------------------------------------------------------------------------------------------
// States per lane and lanes per channel.  All in one lane where the registers take it: 8 states in each of two lanes bring a third wave to a SIMD, but
// every row's own work twice (backward, 16 states: 641 us against 600 at that time).
template <typename F> int by_states(int64_t states, F f) {
  if (states <= 8) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
  if (states <= 16) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
  if (states <= 32) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 2>());
  return f(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
}

int64_t tiles_of(const ppn_scan_args* a) {
  int64_t lanes = 1;
  by_states(a->states, [&](auto, auto lpc) { return (int)(lanes = decltype(lpc)::value); });
  return ceil_div(a->channels / a->groups, 64 / lanes);
}

int64_t states_of(const ppn_scan_args* a) {
  int64_t states = 0;
  by_states(a->states, [&](auto ns, auto lpc) { return (int)(states = decltype(ns)::value * decltype(lpc)::value); });
  return states;
}

// Chunks of time that are worked on at once: one while the waves of (environment, tile) alone fill the chip, since splitting walks the rows
// twice; else as many as bring `wanted` waves, of at least 16 rows.  Forward 3200 (2 x 8724 rows
// x 768: 137, 153, 138 and 142 us at 2000, 2600, 3200 and 4000; 75 x 167 rows x 200: 54, 54, 53, 53), backward 4096 (the latter: 107, 103, 96 us at
// 1024, 2048, 4096).
struct Split { int64_t chunk, chunks; };
// Up to this many chunks, each wave joins the ones before its own by itself, else a launch in between does (75 x 167 rows x 200, 11 chunks: a training step
// takes 194 us against 202, its kernels 156 either way).
constexpr int64_t FEW_CHUNKS = 16;
Split split_time(const ppn_scan_args* a, int64_t waves, int64_t wanted) {
  int64_t chunks = waves * 2 > wanted ? 1 : ceil_div(wanted, waves < 1 ? 1 : waves);
  int64_t chunk = ceil_div(ceil_div(a->time, chunks), ROWS) * ROWS;
  if (chunk < 16) chunk = 16;
  if (ceil_div(a->time, chunk) > 65535) chunk = ceil_div(ceil_div(a->time, 65535), ROWS) * ROWS;
  chunks = a->time ? ceil_div(a->time, chunk) : 1;
  return {chunk, chunks < 1 ? 1 : chunks};
}
Split forward_split(const ppn_scan_args* a) { return split_time(a, a->batch * a->groups * tiles_of(a), 3200); }

struct BackwardPlan { Split split; int64_t rows_bytes, params_bytes, ends_bytes, sums_bytes; };
BackwardPlan plan_backward(const ppn_scan_args* a) {
  BackwardPlan p;
  p.split = split_time(a, a->batch * a->groups * tiles_of(a), 4096);
  auto round = [](int64_t v) { return (v + 255) / 256 * 256; };
  const int64_t cells = a->batch * p.split.chunks;
  p.rows_bytes = round(tiles_of(a) * a->batch * a->time * a->groups * 2 * states_of(a) * 4);
  p.params_bytes = round(cells * (a->states + 2) * a->channels * 4);
  p.ends_bytes = p.split.chunks > 1 ? round(cells * a->states * a->channels * 4) : 0;
  p.sums_bytes = p.split.chunks > 1 ? round(cells * 2 * a->channels * 4) : 0;
  return p;
}

int check(const ppn_scan_args* a) {
  if (!a || a->struct_bytes != (int64_t)sizeof *a) return fail(PPN_E_INVALID, "ppn_scan_args: struct_bytes does not match this library");
  if (a->type < 0 || a->type > PPN_T_F16) return fail(PPN_E_INVALID, "element type %lld is unknown", (long long)a->type);
  if (a->batch < 0 || a->time < 0 || a->channels < 1 || a->groups < 1 || a->channels % a->groups)
    return fail(PPN_E_INVALID, "scan: batch, time >= 0 and channels a multiple of groups >= 1 are needed");
  if (a->batch > 0x7fffffff || a->time > 0x7fffffff || a->channels > (1 << 22)) return fail(PPN_E_INVALID, "scan: a size is out of range");
  const int64_t strides[] = {a->x_time, a->dt_time, a->B_time, a->C_time, a->z_time, a->y_time, a->dy_time, a->dx_time, a->ddt_time, a->dz_time, a->groups * 128};
  for (int64_t v : strides)
    if (v < 0 || v > (1 << 27)) return fail(PPN_E_INVALID, "scan: rows of time may be at most 2^27 elements apart, got %lld", (long long)v);
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
  if (too_many(waves, 64) || (s.chunks > FEW_CHUNKS && too_many(ceil_div(cells, 64), 64)))
    return fail(PPN_E_INVALID, "scan: too many channels of too many environments");
  const dim3 grid(waves, s.chunks);
  float* ends = (float*)a->workspace;
  float* sums = ends + cells * s.chunks;
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return by_states(a->states, [&](auto ns, auto lpc) {
      constexpr int NS = decltype(ns)::value, LPC = decltype(lpc)::value;
      if (s.chunks > 1) {
        scan_forward<T, NS, LPC, SUMMARY><<<grid, dim3(64), 0, (hipStream_t)stream>>>(*a, s.chunk, s.chunks, nullptr, ends, sums);
        if (s.chunks > FEW_CHUNKS) scan_join<false><<<dim3(ceil_div(cells, 64)), dim3(64), 0, (hipStream_t)stream>>>(*a, s.chunks, ends, sums);
      }
      const float* joined = s.chunks > FEW_CHUNKS ? ends : nullptr;
      float* apart = s.chunks > 1 && s.chunks <= FEW_CHUNKS ? ends : nullptr;
      if (a->checkpoints) scan_forward<T, NS, LPC, TRAIN><<<grid, dim3(64), 0, (hipStream_t)stream>>>(*a, s.chunk, s.chunks, joined, apart, sums);
      else scan_forward<T, NS, LPC, OUTPUT><<<grid, dim3(64), 0, (hipStream_t)stream>>>(*a, s.chunk, s.chunks, joined, apart, sums);
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
  const int64_t waves = a->batch * a->groups * tiles_of(a), cells = a->batch * a->states * a->channels, count = a->batch * a->time * a->groups * 2 * states_of(a);
  const int64_t row_blocks = ceil_div(count, 1024), blocks = row_blocks + ceil_div((a->states + 2) * a->channels, 32);
  if (too_many(waves, 64) || (p.split.chunks > FEW_CHUNKS && too_many(ceil_div(cells, 64), 64)) || too_many(blocks, 256))
    return fail(PPN_E_INVALID, "scan: too many rows");
  const dim3 grid(waves, p.split.chunks);
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return by_states(a->states, [&](auto ns, auto lpc) {
      constexpr int NS = decltype(ns)::value, LPC = decltype(lpc)::value;
      const float* joined = p.split.chunks > FEW_CHUNKS ? ends : nullptr;
      if (p.split.chunks > 1) {
        scan_backward<T, NS, LPC, ENDS><<<grid, dim3(64), 0, (hipStream_t)stream>>>(*a, p.split.chunk, p.split.chunks, nullptr, ends, sums, nullptr, nullptr);
        if (joined) scan_join<true><<<dim3(ceil_div(cells, 64)), dim3(64), 0, (hipStream_t)stream>>>(*a, p.split.chunks, ends, sums);
      }
      if (p.split.chunks > 1 && !joined)
        scan_backward<T, NS, LPC, JOINING><<<grid, dim3(64), 0, (hipStream_t)stream>>>(*a, p.split.chunk, p.split.chunks, nullptr, ends, sums, rows, params);
      else
        scan_backward<T, NS, LPC, GRADIENTS><<<grid, dim3(64), 0, (hipStream_t)stream>>>(*a, p.split.chunk, p.split.chunks, joined, nullptr, nullptr, rows, params);
      const ReduceArgs r = {rows, tiles_of(a), a->batch * a->time * a->groups, params, a->batch * p.split.chunks, a->states, a->channels, a->dB, a->dC, a->dA, a->dD,
                            a->ddt_bias, row_blocks};
      scan_reduce<T, NS * LPC><<<dim3(blocks), dim3(256), 0, (hipStream_t)stream>>>(r);
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
  if (a->env_ids && a->rows > MOST_IDS) return fail(PPN_E_INVALID, "ppn_scan_step: at most %d rows with env_ids", MOST_IDS);
  if (a->rows == 0) return PPN_OK;
  if (!a->x || !a->dt || !a->A || !a->B || !a->C || !a->y || !a->state || !a->environments) return fail(PPN_E_INVALID, "ppn_scan_step: x, dt, A, B, C, state (of one environment at least) and y are needed");
  if (too_many(a->rows, 256)) return fail(PPN_E_INVALID, "ppn_scan_step: too many rows");
  const int64_t four = 4 * size_of(a->type);
  const bool wide = a->states % 4 == 0 && aligned(a->state, 16) && aligned(a->A, 16) && aligned(a->B, four) && aligned(a->C, four) && a->B_row % 4 == 0 &&
                    a->C_row % 4 == 0 && a->B_group % 4 == 0 && a->C_group % 4 == 0;
  int lpc = 1;
  while (lpc * 4 < a->states) lpc *= 2;
  // Four channels a lane in flight and at most 4096 workgroups, so that a row's ids are compared by one or a few of them (4096 rows of 512 x 16
  // states out of memory: 72 us, 76 with two workgroups a row); one channel a lane where that leaves less than one workgroup a CU.
  const int64_t per = 256 / lpc;
  const bool few = a->rows * ceil_div(a->channels, 4 * per) < 256;
  int64_t y = ceil_div(a->channels, few ? per : 4 * per);
  if (!few && a->rows * y > 4096) y = ceil_div(4096, a->rows);
  if (y > 65535) y = 65535;
  const dim3 grid(a->rows, y);
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    auto go = [&](auto l) {
      constexpr int LPC = decltype(l)::value;
      if (wide && few) scan_step<T, LPC, true, 1><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a);
      else if (wide) scan_step<T, LPC, true, 4><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a);
      else if (few) scan_step<T, LPC, false, 1><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a);
      else scan_step<T, LPC, false, 4><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a);
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
