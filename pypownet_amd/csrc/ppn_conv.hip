// ppn_conv.hip -- the short causal convolution of a policy's memory: whole windows, their gradients, single rows.
//
// All three are bound by memory: 2 * taps multiply-adds per element against two elements moved (five in a training step).
// A lane owns four neighbouring channels (one where rows are not aligned for that) and walks a stretch of time with the taps - 1 rows
// before it in registers, so every row is read once; neighbouring lanes read neighbouring channels, a wave 512 B or 1 KB at a time.  A row marked in
// `starts` empties the registers.  A window of 1024 x 60 rows of 1024 bfloat16 channels: forward 47 us (252 MB at 5.3 TB/s), backward 89 us (378 MB at
// 4.3 TB/s) and 7 us for the sums; a large copy runs at 4.9 TB/s.
#include "ppn_policy.h"

#include <stdarg.h>
#include <stdio.h>

namespace ppn_policy {

static thread_local char error_text[512];

int fail(int code, const char* format, ...) {
  va_list list;
  va_start(list, format);
  vsnprintf(error_text, sizeof error_text, format, list);
  va_end(list);
  return code;
}

int launched(const char* what) {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? PPN_OK : fail(PPN_E_HIP, "%s: %s", what, hipGetErrorString(e));
}

namespace {

// VEC channels of a row as they are in memory: one load.
template <typename T, int VEC> struct alignas(VEC * sizeof(T)) Raw { T v[VEC]; };

template <typename T, int VEC> __device__ inline void widen(const Raw<T, VEC>& r, float (&out)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = to_float(r.v[i]);
}
template <typename T, int VEC> __device__ inline void load_row(const T* p, float (&out)[VEC]) { widen<T, VEC>(*(const Raw<T, VEC>*)p, out); }
template <typename T, int VEC> __device__ inline void store_row(T* p, const float (&in)[VEC]) {
  Raw<T, VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r.v[i] = (T)in[i];
  *(Raw<T, VEC>*)p = r;
}

// A workgroup of 256 lanes: `width` lanes (whole waves) across the channels, the others on further items.  So a wave is on one environment and
// stretch of time: addresses of rows, flags and episode bookkeeping are scalar, a lane adds its channel as a 32-bit offset.
__host__ __device__ inline int slab_width(int64_t lanes) { return lanes <= 64 ? 64 : lanes <= 128 ? 128 : 256; }
template <typename T, int VEC> __device__ inline Raw<T, VEC> raw_at(const T* row, unsigned lane) { return *(const Raw<T, VEC>*)((const char*)row + lane); }
template <typename T, int VEC> __device__ inline void store_at(T* row, unsigned lane, const float (&in)[VEC]) { store_row<T, VEC>((T*)((char*)row + lane), in); }

// The rows in front of row t0: t0 - 1 is prev[0].  Rows of an earlier episode are zero.
template <typename T, int K, int VEC>
__device__ inline void window_before(const ppn_conv_args& a, int64_t b, int64_t t0, int64_t d, float (&prev)[K - 1][VEC]) {
  const T* x = (const T*)a.x + b * a.x_batch + d;
  const T* first = (const T*)a.initial;
  bool same = true;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    int64_t t = t0 - 1 - j;
    if (same && t >= 0) load_row<T, VEC>(x + t * a.x_time, prev[j]);
    else if (same && first) load_row<T, VEC>(first + (b * (K - 1) + (K - 1 + t)) * a.channels + d, prev[j]);
    else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) prev[j][i] = 0.0f;
    }
    if (a.starts && t >= 0 && a.starts[b * a.starts_batch + t * a.starts_time]) same = false;
  }
}

template <int K, int VEC> __device__ inline void clear(float (&rows)[K][VEC]) {
#pragma unroll
  for (int j = 0; j < K; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) rows[j][i] = 0.0f;
}

template <int K, int VEC> __device__ inline void load_weights(const float* weight, const float* bias, int64_t d, float (&w)[K][VEC], float (&c)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][i] = weight[(d + i) * K + k];
    c[i] = bias ? bias[d + i] : 0.0f;
  }
}

// One lane: VEC channels of one environment over `span` rows.  Blocks of AHEAD rows: the next block's loads are issued before this block's
// stores, and no branch of the loop holds a memory operation, so that waiting for the loads is not waiting for the stores.
template <typename T, int K, int VEC>
__global__ void __launch_bounds__(256) conv_forward(ppn_conv_args a, int64_t span, int stretches) {
  const int lanes = (int)(a.channels / VEC), width = slab_width(lanes), depth = 256 / width;
  const int deep = __builtin_amdgcn_readfirstlane(threadIdx.x / width), item = blockIdx.x * depth + deep;
  if (item >= a.batch * stretches) return;
  // (a lane past the last channel does the last one's work again: all lanes of a wave take part in its episode bookkeeping)
  const int cv = min((int)(blockIdx.y * width + threadIdx.x % width), lanes - 1);
  const int64_t d = cv * VEC, b = item / stretches, t0 = (item - b * stretches) * span;
  const int64_t t1 = t0 + span < a.time ? t0 + span : a.time;
  const unsigned lane = (unsigned)d * (unsigned)sizeof(T);
  float w[K][VEC], c[VEC], prev[K - 1][VEC];
  load_weights<K, VEC>(a.weight, a.bias, d, w, c);
  window_before<T, K, VEC>(a, b, t0, d, prev);
  const T* x = (const T*)a.x + b * a.x_batch;
  T* y = (T*)a.y + b * a.y_batch + t0 * a.y_time;
  const uint8_t* starts = a.starts ? a.starts + b * a.starts_batch : nullptr;
  const bool silu = a.silu;
  constexpr int AHEAD = 4;
  Raw<T, VEC> next[AHEAD];
  unsigned nflag = 0;                       // lane j of the wave: the flag of the next block's row j
  const int wave_lane = (threadIdx.x & 63) < AHEAD ? threadIdx.x & 63 : AHEAD - 1;
  auto fetch = [&](int64_t t) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int64_t at = t + j < t1 ? t + j : t1 - 1;
      next[j] = raw_at<T, VEC>(x + at * a.x_time, lane);
    }
    if (starts) nflag = starts[(t + wave_lane < t1 ? t + wave_lane : t1 - 1) * a.starts_time];
  };
  auto step = [&](const Raw<T, VEC>& raw, bool begins) {
    __builtin_amdgcn_sched_barrier(0);      // (rows one after the other: mixing them takes registers, that is waves)
    float row[VEC], out[VEC];
    widen<T, VEC>(raw, row);
    if (begins) clear<K - 1, VEC>(prev);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float s = c[i] + w[K - 1][i] * row[i];
#pragma unroll
      for (int k = 0; k < K - 1; ++k) s += w[K - 2 - k][i] * prev[k][i];
      out[i] = silu ? s * sigmoid(s) : s;
    }
    store_at<T, VEC>(y, lane, out);
    y += a.y_time;
#pragma unroll
    for (int k = K - 2; k > 0; --k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) prev[k][i] = prev[k - 1][i];
#pragma unroll
    for (int i = 0; i < VEC; ++i) prev[0][i] = row[i];
  };
  if (t0 < t1) fetch(t0);
  int64_t t = t0;
  for (; t + AHEAD <= t1; t += AHEAD) {
    Raw<T, VEC> row[AHEAD];
    const unsigned begins = (unsigned)__ballot(nflag != 0);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) row[j] = next[j];
    fetch(t + AHEAD);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) step(row[j], (begins >> j) & 1);
  }
  const unsigned begins = (unsigned)__ballot(nflag != 0);
#pragma unroll
  for (int j = 0; j < AHEAD - 1; ++j)
    if (t + j < t1) step(next[j], (begins >> j) & 1);
  if (t1 == a.time && a.final_state) {
    T* last = (T*)a.final_state + b * (K - 1) * a.channels;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) store_at<T, VEC>(last + (K - 2 - k) * a.channels, lane, prev[k]);
  }
}

// Backward.  With s = the sum in front of the activation and g = dy act'(s):
//   dx[t] = sum_j weight[K-1-j] g[t+j]   over the rows t..t+K-1 of t's episode,   dweight[k] = sum g[t] x[t-K+1+k],   dbias = sum g.
// A lane recomputes s walking forward (K - 1 rows past its stretch too, for the dx of its last rows) with the unfinished dx of the
// last K - 1 rows in registers.  The sums over rows and environments are kept in registers while the workgroup goes over its
// share of the (environment, stretch) items, added up over the workgroup's lanes of equal channel in LDS and left as one row of
// partial sums per workgroup; conv_reduce adds those rows in a fixed order, so a gradient is the same in every run.
template <typename T, int K, int VEC>
__global__ void __launch_bounds__(256) conv_backward(ppn_conv_args a, int64_t span, int stretches, float* partial) {
  // grid.x: slabs of `width` lanes across the channels, grid.y: shares of the items; a workgroup takes 256 / width items at a time
  const int lanes = (int)(a.channels / VEC), width = slab_width(lanes), depth = 256 / width;
  const int deep = __builtin_amdgcn_readfirstlane(threadIdx.x / width), cv = blockIdx.x * width + threadIdx.x % width;
  const bool live = cv < lanes, silu = a.silu;
  const int64_t d = min(cv, lanes - 1) * VEC;      // (a lane past the last channel does the last one's work again, but leaves no sums)
  const int items = (int)(a.batch * stretches);
  const unsigned lane = (unsigned)d * (unsigned)sizeof(T);
  float w[K][VEC], c[VEC], dw[K][VEC], db[VEC];
  load_weights<K, VEC>(a.weight, a.bias, d, w, c);
  clear<K, VEC>(dw);
#pragma unroll
  for (int i = 0; i < VEC; ++i) db[i] = 0.0f;
  for (int item = blockIdx.y * depth + deep; item < items; item += gridDim.y * depth) {
    const int64_t b = item / stretches, t0 = (item - b * stretches) * span;
    const int64_t t1 = t0 + span < a.time ? t0 + span : a.time, reach = t1 + K - 1 < a.time ? t1 + K - 1 : a.time;
    const T* x = (const T*)a.x + b * a.x_batch;
    const T* dy = (const T*)a.dy + b * a.dy_batch;
    T* dx = (T*)a.dx + b * a.dx_batch;
    T* dfirst = (T*)a.dinitial + b * (K - 1) * a.channels;
    const uint8_t* starts = a.starts ? a.starts + b * a.starts_batch : nullptr;
    float prev[K - 1][VEC], open[K - 1][VEC];   // open[j]: dx of row t - 1 - j, still to receive
    window_before<T, K, VEC>(a, b, t0, d, prev);
    clear<K - 1, VEC>(open);
    // The first row whose dx is not out yet: the stretch's first (or the first of `initial`), later the first of the running episode.
    int64_t pending = t0 == 0 && a.dinitial ? -(K - 1) : t0;
    auto row_of_dx = [&](int64_t at) { return at < 0 ? dfirst + (K - 1 + at) * a.channels : dx + at * a.dx_time; };
    constexpr int AHEAD = 4;
    Raw<T, VEC> nrow[AHEAD], nup[AHEAD];
    unsigned nflag = 0;                       // lane j of the wave: the flag of the next block's row j
    const int wave_lane = (threadIdx.x & 63) < AHEAD ? threadIdx.x & 63 : AHEAD - 1;
    auto fetch = [&](int64_t t) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int64_t at = t + j < reach ? t + j : reach - 1;
        nrow[j] = raw_at<T, VEC>(x + at * a.x_time, lane);
        nup[j] = raw_at<T, VEC>(dy + at * a.dy_time, lane);
      }
      if (starts) nflag = starts[(t + wave_lane < reach ? t + wave_lane : reach - 1) * a.starts_time];
    };
    // One row: its part of the dx of the rows t - K + 1 .. t, of which the first is then complete.  A start completes all rows in front of it at once;
    // the row that is out of turn then is written again where the first pending row will be, ahead of that row's own value, so that every
    // row writes one.  inside: row t belongs to this stretch (else to the next, and only its part of this one's dx counts).
    auto step = [&](int64_t t, const Raw<T, VEC>& raw, const Raw<T, VEC>& raw_up, bool begins, bool inside) {
      __builtin_amdgcn_sched_barrier(0);
      float row[VEC], g[VEC];
      widen<T, VEC>(raw, row);
      widen<T, VEC>(raw_up, g);
      if (begins) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
          const int64_t at = t - 1 - k;
          if (at >= pending && at < t1) store_at<T, VEC>(row_of_dx(at), lane, open[k]);
        }
        clear<K - 1, VEC>(open);
        clear<K - 1, VEC>(prev);
        pending = t;
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float s = c[i] + w[K - 1][i] * row[i];
#pragma unroll
        for (int k = 0; k < K - 1; ++k) s += w[K - 2 - k][i] * prev[k][i];
        const float q = sigmoid(s);
        g[i] = silu ? g[i] * q * (1.0f + s * (1.0f - q)) : g[i];
        if (inside) {
          db[i] += g[i];
          dw[K - 1][i] += g[i] * row[i];
#pragma unroll
          for (int k = 0; k < K - 1; ++k) dw[K - 2 - k][i] += g[i] * prev[k][i];
        }
#pragma unroll
        for (int k = 0; k < K - 1; ++k) open[k][i] += g[i] * w[K - 2 - k][i];
      }
      const int64_t first = t - (K - 1), at = first > pending ? first : pending;
      if (inside || at < t1) store_at<T, VEC>(row_of_dx(at), lane, open[K - 2]);
#pragma unroll
      for (int k = K - 2; k > 0; --k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) open[k][i] = open[k - 1][i], prev[k][i] = prev[k - 1][i];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        open[0][i] = g[i] * w[K - 1][i];
        prev[0][i] = row[i];
      }
    };
    int64_t t = t0;
    if (t < reach) fetch(t);
    for (; t + AHEAD <= t1; t += AHEAD) {        // (as in the forward pass: loads ahead, no branch around the memory operations of every row)
      Raw<T, VEC> row[AHEAD], up[AHEAD];
      const unsigned begins = (unsigned)__ballot(nflag != 0);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) row[j] = nrow[j], up[j] = nup[j];
      fetch(t + AHEAD);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) step(t + j, row[j], up[j], (begins >> j) & 1, true);
    }
    for (; t < reach; ++t) {
      fetch(t);
      step(t, nrow[0], nup[0], (unsigned)__ballot(nflag != 0) & 1, t < t1);
    }
    // rows reach - (K - 1) .. reach - 1 are still open: past the end of time the final state's gradient joins those of the last episode
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      const int64_t at = reach - 1 - k;
      if (at < pending || at >= t1) continue;
      if (reach == a.time && a.dfinal) {
        float f[VEC];
        load_row<T, VEC>((const T*)a.dfinal + (b * (K - 1) + (K - 2 - k)) * a.channels + d, f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) open[k][i] += f[i];
      }
      store_at<T, VEC>(row_of_dx(at), lane, open[k]);
    }
  }
  __shared__ float sums[256][VEC + 1];
  float* out = partial + (int64_t)blockIdx.y * (K + 1) * a.channels;
#pragma unroll
  for (int k = 0; k < K + 1; ++k) {
    if (depth > 1) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) sums[threadIdx.x][i] = k < K ? dw[k < K ? k : 0][i] : db[i];
      __syncthreads();
    }
    if (deep == 0 && live) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float s = k < K ? dw[k < K ? k : 0][i] : db[i];
        for (int q = 1; q < depth; ++q) s += sums[q * width + threadIdx.x][i];
        out[k * a.channels + d + i] = s;
      }
    }
    if (depth > 1) __syncthreads();
  }
}

// Adds the workgroups' partial rows [shares x (K + 1) x channels]: 32 columns a workgroup, 16 lanes a column (1024 shares of 5 x 1024: 7 us, 12 with
// 8).
constexpr int REDUCE_PARTS = 16;
__global__ void __launch_bounds__(32 * REDUCE_PARTS) conv_reduce(const float* partial, int64_t shares, int64_t channels, int64_t taps, float* dweight, float* dbias) {
  const int64_t columns = (taps + 1) * channels, col = (int64_t)blockIdx.x * 32 + threadIdx.x % 32;
  const int part = threadIdx.x / 32;
  float s = 0.0f;
  if (col < columns)
    for (int64_t r = part; r < shares; r += 8 * REDUCE_PARTS) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = partial[(r + REDUCE_PARTS * i < shares ? r + REDUCE_PARTS * i : r) * columns + col];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += r + REDUCE_PARTS * i < shares ? v[i] : 0.0f;
    }
  __shared__ float sums[REDUCE_PARTS][33];
  sums[part][threadIdx.x % 32] = s;
  __syncthreads();
  if (part == 0 && col < columns) {
    for (int q = 1; q < REDUCE_PARTS; ++q) s += sums[q][threadIdx.x];
    const int64_t k = col / channels, d = col - k * channels;
    if (k < taps) dweight[d * taps + k] = s;
    else if (dbias) dbias[d] = s;
  }
}

template <typename T, int K, int VEC>
__global__ void __launch_bounds__(256) conv_step(ppn_conv_step_args a) {
  const int64_t row = blockIdx.x, lanes = a.channels / VEC, cv = (int64_t)blockIdx.y * 256 + threadIdx.x, d = (cv < lanes ? cv : lanes - 1) * VEC;
  T* window = (T*)a.state + row_env(a.env_ids, row, a.environments) * (K - 1) * a.channels + d;
  T* y = (T*)a.y + row * a.y_row + d;
  float w[K][VEC], c[VEC], rows[K][VEC], out[VEC];
  const bool begins = a.starts && a.starts[row];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) load_row<T, VEC>(window + k * a.channels, rows[k]);
  load_row<T, VEC>((const T*)a.x + row * a.x_row + d, rows[K - 1]);
  load_weights<K, VEC>(a.weight, a.bias, d, w, c);
  const int live = row_state(a.env_ids, row, a.environments);      // (the loads are under way while the ids are compared)
  if (cv >= lanes) return;
  if (begins) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) rows[k][i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float s = c[i] + w[K - 1][i] * rows[K - 1][i];           // (conv_forward's order: a window read row by row gives the same bits)
#pragma unroll
    for (int k = K - 2; k >= 0; --k) s += w[k][i] * rows[k][i];
    out[i] = live == ROW_LIVE ? (a.silu ? s * sigmoid(s) : s) : live == ROW_PADDING ? 0.0f : __builtin_nanf("");
  }
  store_row<T, VEC>(y, out);
  if (live != ROW_LIVE) return;
#pragma unroll
  for (int k = 0; k < K - 1; ++k) store_row<T, VEC>(window + k * a.channels, rows[k + 1]);
}

template <typename F> int by_taps(int64_t taps, F f) {
  switch (taps) {
    case 2: return f(std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, 3>());
    case 4: return f(std::integral_constant<int, 4>());
    case 5: return f(std::integral_constant<int, 5>());
    case 6: return f(std::integral_constant<int, 6>());
    case 7: return f(std::integral_constant<int, 7>());
    case 8: return f(std::integral_constant<int, 8>());
  }
  return fail(PPN_E_INVALID, "taps must be 2..8, got %lld", (long long)taps);
}

int check(const ppn_conv_args* a) {
  if (!a || a->struct_bytes != (int64_t)sizeof *a) return fail(PPN_E_INVALID, "ppn_conv_args: struct_bytes does not match this library");
  if (a->batch < 0 || a->time < 0 || a->channels < 1) return fail(PPN_E_INVALID, "convolution: batch, time >= 0 and channels >= 1 are needed");
  if (a->batch > 0x7fffffff || a->time > 0x7fffffff || a->channels > (1 << 22)) return fail(PPN_E_INVALID, "convolution: a size is out of range");
  if (a->taps < 2 || a->taps > 8) return fail(PPN_E_INVALID, "taps must be 2..8, got %lld", (long long)a->taps);
  if (a->type < 0 || a->type > PPN_T_F16) return fail(PPN_E_INVALID, "element type %lld is unknown", (long long)a->type);
  return PPN_OK;
}

// Four channels a lane (16 bytes, or 8 of the 16-bit types: eight channels' weights, sums and rows would leave half the waves) where they fill a wave
// and every row of every tensor begins on such a border; else one.  A wave of fewer channels does some of them twice.  One against four channels a lane,
// forward and training step of 63 million elements in bfloat16, in us: 53 and 111, 195 and 394 at 64 channels; 48 and 59, 193 and 218 at 128; 61 and
// 47, 245 and 176 at 192 (left to one, as 32 bits is even: 102 and 102, 277 and 269).  In 32 bits at 128 channels: 111 and 110, 299 and 283.
constexpr int WIDE = 4;
bool wide(const ppn_conv_args* a, bool backward) {
  const int64_t vec = WIDE, bytes = WIDE * size_of(a->type);
  if (a->channels < 64 * WIDE) return false;
  const bool b = a->batch > 1, t = a->time > 1;      // (a stride that is never taken does not matter)
  const int64_t strides[] = {a->channels, b * a->x_batch, t * a->x_time, b * (backward ? a->dy_batch : a->y_batch), t * (backward ? a->dy_time : a->y_time),
                             backward ? b * a->dx_batch : 0, backward ? t * a->dx_time : 0};
  for (int64_t s : strides)
    if (s % vec) return false;
  const void* bases[] = {a->x, a->initial, backward ? a->dy : a->y, backward ? a->dx : a->final_state, backward ? a->dfinal : nullptr,
                         backward ? a->dinitial : nullptr};
  for (const void* p : bases)
    if (!aligned(p, bytes)) return false;
  return true;
}

// Rows per lane: as many as leave the chip `wanted` lanes, at least 16 (a stretch reads taps - 1 rows of its neighbour again).
int64_t span_for(int64_t batch, int64_t time, int64_t lanes, int64_t wanted) {
  int64_t stretches = ceil_div(wanted, batch * lanes > 0 ? batch * lanes : 1);
  int64_t span = ceil_div(time, stretches < 1 ? 1 : stretches);
  if (span < 16) span = 16;
  return span < time ? span : time;
}

struct BackwardPlan { int64_t vec, lanes, span, stretches, slabs, shares; };

BackwardPlan plan_backward(const ppn_conv_args* a) {
  BackwardPlan p;
  p.vec = wide(a, true) ? WIDE : 1;
  p.lanes = a->channels / p.vec;
  p.span = span_for(a->batch, a->time, p.lanes, 131072);
  if (p.span < 1) p.span = 1;
  p.stretches = a->time ? ceil_div(a->time, p.span) : 1;      // (no rows at all: the final state's gradient still passes to `initial`)
  const int64_t width = slab_width(p.lanes), depth = 256 / width;
  p.slabs = ceil_div(p.lanes, width);
  // 1024 workgroups in all: four for each CU, and few enough partial rows (shares x (taps + 1) x channels floats)
  p.shares = ceil_div(1024, p.slabs);
  const int64_t most = ceil_div(a->batch * p.stretches, depth);
  if (p.shares > most) p.shares = most;
  if (p.shares < 1) p.shares = 1;
  return p;
}

}  // namespace
}  // namespace ppn_policy

using namespace ppn_policy;

extern "C" const char* ppn_policy_error(void) { return error_text; }

extern "C" int ppn_conv_forward(const ppn_conv_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  if (!a->x || !a->weight || !a->y) {
    if (a->batch * a->time) return fail(PPN_E_INVALID, "ppn_conv_forward: x, weight and y are needed");
  }
  if (a->batch == 0) return PPN_OK;
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return by_taps(a->taps, [&](auto k) {
      constexpr int K = decltype(k)::value;
      const bool w = wide(a, false);
      const int64_t lanes = a->channels / (w ? WIDE : 1);
      const int64_t span = a->time ? span_for(a->batch, a->time, lanes, 131072) : 1, stretches = a->time ? ceil_div(a->time, span) : 1;
      const int64_t width = slab_width(lanes);
      if (too_many(ceil_div(a->batch * stretches, 256 / width), 256)) return fail(PPN_E_INVALID, "convolution: too many environments");
      const dim3 grid(ceil_div(a->batch * stretches, 256 / width), ceil_div(lanes, width));
      if (w) conv_forward<T, K, WIDE><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a, span, (int)stretches);
      else conv_forward<T, K, 1><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a, span, (int)stretches);
      return launched("ppn_conv_forward");
    });
  });
}

extern "C" int64_t ppn_conv_backward_workspace(const ppn_conv_args* a) {
  if (int rc = check(a)) return rc;
  return plan_backward(a).shares * (a->taps + 1) * a->channels * 4;
}

extern "C" int ppn_conv_backward(const ppn_conv_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  if (!a->weight || !a->dweight || !a->workspace) return fail(PPN_E_INVALID, "ppn_conv_backward: weight, dweight and a workspace are needed");
  if (a->batch * a->time && (!a->x || !a->dy || !a->dx)) return fail(PPN_E_INVALID, "ppn_conv_backward: x, dy and dx are needed");
  const BackwardPlan p = plan_backward(a);
  if (a->workspace_bytes < p.shares * (a->taps + 1) * a->channels * 4) return fail(PPN_E_INVALID, "ppn_conv_backward: the workspace is too small");
  if (a->batch * p.stretches > 0x7fff0000) return fail(PPN_E_INVALID, "convolution: too many environments");
  if (p.shares > 65535) return fail(PPN_E_INVALID, "ppn_conv_backward: too many shares");
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return by_taps(a->taps, [&](auto k) {
      constexpr int K = decltype(k)::value;
      const dim3 grid(p.slabs, p.shares);
      if (p.vec > 1) conv_backward<T, K, WIDE><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a, p.span, (int)p.stretches, (float*)a->workspace);
      else conv_backward<T, K, 1><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a, p.span, (int)p.stretches, (float*)a->workspace);
      conv_reduce<<<dim3(ceil_div((K + 1) * a->channels, 32)), dim3(32 * REDUCE_PARTS), 0, (hipStream_t)stream>>>((const float*)a->workspace, p.shares, a->channels, K,
                                                                                                   a->dweight, a->dbias);
      return launched("ppn_conv_backward");
    });
  });
}

extern "C" int ppn_conv_step(const ppn_conv_step_args* a, void* stream) {
  if (!a || a->struct_bytes != (int64_t)sizeof *a) return fail(PPN_E_INVALID, "ppn_conv_step_args: struct_bytes does not match this library");
  if (a->rows < 0 || a->environments < 0 || a->channels < 1 || a->channels > (1 << 24) || a->rows > 0x7fffffff)
    return fail(PPN_E_INVALID, "ppn_conv_step: a size is out of range");
  if (!a->env_ids && a->rows > a->environments) return fail(PPN_E_INVALID, "ppn_conv_step: more rows than environments and no env_ids");
  if (a->env_ids && a->rows > MOST_IDS) return fail(PPN_E_INVALID, "ppn_conv_step: at most %d rows with env_ids", MOST_IDS);
  if (a->rows == 0) return PPN_OK;
  if (!a->x || !a->weight || !a->y || !a->state || !a->environments) return fail(PPN_E_INVALID, "ppn_conv_step: x, weight, state (of one environment at least) and y are needed");
  const int64_t vec = WIDE, bytes = WIDE * size_of(a->type);
  const bool w = a->channels % vec == 0 && a->x_row % vec == 0 && a->y_row % vec == 0 && aligned(a->x, bytes) && aligned(a->y, bytes) && aligned(a->state, bytes);
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return by_taps(a->taps, [&](auto k) {
      constexpr int K = decltype(k)::value;
      const dim3 grid(a->rows, ceil_div(a->channels / (w ? vec : 1), 256));
      if (grid.y > 65535) return fail(PPN_E_INVALID, "ppn_conv_step: too many channels");
      if (too_many(a->rows, 256)) return fail(PPN_E_INVALID, "ppn_conv_step: too many rows");
      if (w) conv_step<T, K, WIDE><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a);
      else conv_step<T, K, 1><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a);
      return launched("ppn_conv_step");
    });
  });
}
