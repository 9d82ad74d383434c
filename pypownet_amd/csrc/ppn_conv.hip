// ppn_conv.hip -- the short causal convolution of a policy's memory: whole windows, their gradients, single rows.
//
// All three are bound by memory: 2 * taps multiply-adds per element against two elements moved (five in a training step).
// A lane owns VEC neighbouring channels (16 bytes, or one channel where rows are not 16-byte aligned) and walks a stretch of
// time with the taps - 1 rows before it in registers, so every row is read once; neighbouring lanes read neighbouring
// channels, a wave 1 KB at a time.  A row marked in `starts` empties the registers.
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

template <typename T, int VEC> __device__ inline void load_row(const T* p, float (&out)[VEC]) {
  if constexpr (VEC == 1) {
    out[0] = to_float(p[0]);
  } else {
    Pack<T> k = *(const Pack<T>*)p;
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = to_float(k.v[i]);
  }
}

template <typename T, int VEC> __device__ inline void store_row(T* p, const float (&in)[VEC]) {
  if constexpr (VEC == 1) {
    p[0] = (T)in[0];
  } else {
    Pack<T> k;
#pragma unroll
    for (int i = 0; i < VEC; ++i) k.v[i] = (T)in[i];
    *(Pack<T>*)p = k;
  }
}

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

// One lane: VEC channels of one environment over `span` rows.  Lanes are numbered (environment, stretch, channel) with the channel fastest.
template <typename T, int K, int VEC>
__global__ void __launch_bounds__(256) conv_forward(ppn_conv_args a, int64_t span, int64_t stretches) {
  const int64_t lanes = a.channels / VEC;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t item = id / lanes;
  if (item >= a.batch * stretches) return;
  const int64_t d = (id - item * lanes) * VEC, b = item / stretches, t0 = (item - b * stretches) * span;
  const int64_t t1 = t0 + span < a.time ? t0 + span : a.time;
  float w[K][VEC], c[VEC], prev[K - 1][VEC];
  load_weights<K, VEC>(a.weight, a.bias, d, w, c);
  window_before<T, K, VEC>(a, b, t0, d, prev);
  const T* x = (const T*)a.x + b * a.x_batch + d;
  T* y = (T*)a.y + b * a.y_batch + d;
  const uint8_t* starts = a.starts ? a.starts + b * a.starts_batch : nullptr;
  constexpr int AHEAD = 4;                       // rows whose loads are in flight together
  for (int64_t t = t0; t < t1; t += AHEAD) {
    float row[AHEAD][VEC];
    bool begins[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      int64_t at = t + j < t1 ? t + j : t1 - 1;
      load_row<T, VEC>(x + at * a.x_time, row[j]);
      begins[j] = starts && starts[at * a.starts_time];
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (t + j >= t1) break;
      if (begins[j]) clear<K - 1, VEC>(prev);
      float out[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float s = c[i] + w[K - 1][i] * row[j][i];
#pragma unroll
        for (int k = 0; k < K - 1; ++k) s += w[K - 2 - k][i] * prev[k][i];
        out[i] = a.silu ? s * sigmoid(s) : s;
      }
      store_row<T, VEC>(y + (t + j) * a.y_time, out);
#pragma unroll
      for (int k = K - 2; k > 0; --k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) prev[k][i] = prev[k - 1][i];
#pragma unroll
      for (int i = 0; i < VEC; ++i) prev[0][i] = row[j][i];
    }
  }
  if (t1 == a.time && a.final_state) {
    T* last = (T*)a.final_state + b * (K - 1) * a.channels + d;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) store_row<T, VEC>(last + (K - 2 - k) * a.channels, prev[k]);
  }
}

// Lanes across the channels of a workgroup of the backward pass; the other lanes take further items.
__host__ __device__ inline int slab_width(int64_t lanes) { return lanes <= 64 ? 64 : lanes <= 128 ? 128 : 256; }

// Backward.  With s = the sum in front of the activation and g = dy act'(s):
//   dx[t] = sum_j weight[K-1-j] g[t+j]   over the rows t..t+K-1 of t's episode,   dweight[k] = sum g[t] x[t-K+1+k],   dbias = sum g.
// A lane recomputes s walking forward (K - 1 rows past its stretch too, for the dx of its last rows) with the unfinished dx of the
// last K - 1 rows in registers.  The sums over rows and environments are kept in registers while the workgroup goes over its
// share of the (environment, stretch) items, added up over the workgroup's lanes of equal channel in LDS and left as one row of
// partial sums per workgroup; conv_reduce adds those rows in a fixed order, so a gradient is the same in every run.
template <typename T, int K, int VEC>
__global__ void __launch_bounds__(256) conv_backward(ppn_conv_args a, int64_t span, int64_t stretches, float* partial) {
  // grid.x: slabs of `width` lanes across the channels, grid.y: shares of the items; a workgroup takes 256 / width items at a time
  const int64_t lanes = a.channels / VEC;
  const int width = slab_width(lanes);
  const int lane = threadIdx.x % width, deep = threadIdx.x / width, depth = 256 / width;
  const int64_t cv = (int64_t)blockIdx.x * width + lane;
  const bool live = cv < lanes;
  const int64_t d = (live ? cv : 0) * VEC, items = a.batch * stretches;
  float w[K][VEC], c[VEC], dw[K][VEC], db[VEC];
  load_weights<K, VEC>(a.weight, a.bias, d, w, c);
  clear<K, VEC>(dw);
#pragma unroll
  for (int i = 0; i < VEC; ++i) db[i] = 0.0f;
  if (live) {
    for (int64_t item = (int64_t)blockIdx.y * depth + deep; item < items; item += (int64_t)gridDim.y * depth) {
      const int64_t b = item / stretches, t0 = (item - b * stretches) * span;
      const int64_t t1 = t0 + span < a.time ? t0 + span : a.time, reach = t1 + K - 1 < a.time ? t1 + K - 1 : a.time;
      const T* x = (const T*)a.x + b * a.x_batch + d;
      const T* dy = (const T*)a.dy + b * a.dy_batch + d;
      T* dx = (T*)a.dx + b * a.dx_batch + d;
      const uint8_t* starts = a.starts ? a.starts + b * a.starts_batch : nullptr;
      float prev[K - 1][VEC], open[K - 1][VEC];   // open[j]: dx of row t - 1 - j, still to receive
      window_before<T, K, VEC>(a, b, t0, d, prev);
      clear<K - 1, VEC>(open);
      int alive = 0;                               // rows in front of t of t's episode (of the stretch, or of `initial` for the first one)
      const bool from_initial = t0 == 0 && a.dinitial;
      if (from_initial) alive = K - 1;
      constexpr int AHEAD = 4;
      for (int64_t tb = t0; tb < reach; tb += AHEAD) {
        float row[AHEAD][VEC], up[AHEAD][VEC];
        bool begins[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          int64_t at = tb + j < reach ? tb + j : reach - 1;
          load_row<T, VEC>(x + at * a.x_time, row[j]);
          load_row<T, VEC>(dy + at * a.dy_time, up[j]);
          begins[j] = starts && starts[at * a.starts_time];
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          const int64_t t = tb + j;
          if (t >= reach) break;
          if (begins[j]) {
            clear<K - 1, VEC>(prev);
            alive = 0;
          }
          const bool inside = t < t1;
          float g[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float s = c[i] + w[K - 1][i] * row[j][i];
#pragma unroll
            for (int k = 0; k < K - 1; ++k) s += w[K - 2 - k][i] * prev[k][i];
            float q = sigmoid(s);
            g[i] = a.silu ? up[j][i] * q * (1.0f + s * (1.0f - q)) : up[j][i];
            if (inside) {
              db[i] += g[i];
              dw[K - 1][i] += g[i] * row[j][i];
            }
          }
#pragma unroll
          for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              if (inside) dw[K - 2 - k][i] += g[i] * prev[k][i];
              if (k < alive) open[k][i] += g[i] * w[K - 2 - k][i];
            }
          // row t - (K - 1) is complete
          const int64_t done = t - (K - 1);
          if (done >= t0) store_row<T, VEC>(dx + done * a.dx_time, open[K - 2]);
          else if (from_initial && done < 0) store_row<T, VEC>((T*)a.dinitial + (b * (K - 1) + (K - 1 + done)) * a.channels + d, open[K - 2]);
#pragma unroll
          for (int k = K - 2; k > 0; --k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) open[k][i] = open[k - 1][i], prev[k][i] = prev[k - 1][i];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            open[0][i] = g[i] * w[K - 1][i];
            prev[0][i] = row[j][i];
          }
          if (alive < K - 1) ++alive;
        }
      }
      // rows reach - (K - 1) .. reach - 1 are still open: past the end of time the final state's gradient joins those of the last episode
      const bool end = reach == a.time;
#pragma unroll
      for (int k = 0; k < K - 1; ++k) {
        const int64_t t = reach - 1 - k;
        if (end && a.dfinal && k < alive) {
          float f[VEC];
          load_row<T, VEC>((const T*)a.dfinal + (b * (K - 1) + (K - 2 - k)) * a.channels + d, f);
#pragma unroll
          for (int i = 0; i < VEC; ++i) open[k][i] += f[i];
        }
        if (t >= t0 && t < t1) store_row<T, VEC>(dx + t * a.dx_time, open[k]);
        else if (from_initial && t < 0) store_row<T, VEC>((T*)a.dinitial + (b * (K - 1) + (K - 1 + t)) * a.channels + d, open[k]);
      }
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
        for (int q = 1; q < depth; ++q) s += sums[q * width + lane][i];
        out[k * a.channels + d + i] = s;
      }
    }
    if (depth > 1) __syncthreads();
  }
}

// Adds the workgroups' partial rows [shares x (K + 1) x channels]: 32 columns a workgroup, 8 lanes a column.
__global__ void __launch_bounds__(256) conv_reduce(const float* partial, int64_t shares, int64_t channels, int64_t taps, float* dweight, float* dbias) {
  const int64_t columns = (taps + 1) * channels, col = (int64_t)blockIdx.x * 32 + threadIdx.x % 32;
  const int part = threadIdx.x / 32;
  float s = 0.0f;
  if (col < columns)
    for (int64_t r = part; r < shares; r += 8) s += partial[r * columns + col];
  __shared__ float sums[8][33];
  sums[part][threadIdx.x % 32] = s;
  __syncthreads();
  if (part == 0 && col < columns) {
    for (int q = 1; q < 8; ++q) s += sums[q][threadIdx.x];
    const int64_t k = col / channels, d = col - k * channels;
    if (k < taps) dweight[d * taps + k] = s;
    else if (dbias) dbias[d] = s;
  }
}

template <typename T, int K, int VEC>
__global__ void __launch_bounds__(256) conv_step(ppn_conv_step_args a) {
  const int64_t row = blockIdx.x, lanes = a.channels / VEC;
  const int64_t cv = (int64_t)blockIdx.y * 256 + threadIdx.x;
  const int64_t d = cv * VEC;
  const int state = row_state(a.env_ids, row, a.environments);
  if (cv >= lanes) return;
  T* y = (T*)a.y + row * a.y_row + d;
  float out[VEC];
  if (state != ROW_LIVE) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = state == ROW_PADDING ? 0.0f : __builtin_nanf("");
    store_row<T, VEC>(y, out);
    return;
  }
  const int64_t env = a.env_ids ? a.env_ids[row] : row;
  T* window = (T*)a.state + env * (K - 1) * a.channels + d;
  float w[K][VEC], c[VEC], rows[K][VEC];
  const bool begins = a.starts && a.starts[row];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) {
    load_row<T, VEC>(window + k * a.channels, rows[k]);
    if (begins) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) rows[k][i] = 0.0f;
    }
  }
  load_row<T, VEC>((const T*)a.x + row * a.x_row + d, rows[K - 1]);
  load_weights<K, VEC>(a.weight, a.bias, d, w, c);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float s = c[i] + w[K - 1][i] * rows[K - 1][i];           // (conv_forward's order: a window read row by row gives the same bits)
#pragma unroll
    for (int k = K - 2; k >= 0; --k) s += w[k][i] * rows[k][i];
    out[i] = a.silu ? s * sigmoid(s) : s;
  }
  store_row<T, VEC>(y, out);
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
  if (a->batch > 0x7fffffff || a->time > 0x7fffffff || a->channels > (1 << 24)) return fail(PPN_E_INVALID, "convolution: a size is out of range");
  if (a->taps < 2 || a->taps > 8) return fail(PPN_E_INVALID, "taps must be 2..8, got %lld", (long long)a->taps);
  if (a->type < 0 || a->type > PPN_T_F16) return fail(PPN_E_INVALID, "element type %lld is unknown", (long long)a->type);
  return PPN_OK;
}

// 16-byte rows: every row of every tensor begins on a 16-byte border.
bool wide(const ppn_conv_args* a, bool backward) {
  const int64_t vec = 16 / size_of(a->type);
  const int64_t strides[] = {a->channels, a->x_batch, a->x_time, backward ? a->dy_batch : a->y_batch, backward ? a->dy_time : a->y_time,
                             backward ? a->dx_batch : 0, backward ? a->dx_time : 0};
  for (int64_t s : strides)
    if (s % vec) return false;
  const void* bases[] = {a->x, a->initial, backward ? a->dy : a->y, backward ? a->dx : a->final_state, backward ? a->dfinal : nullptr,
                         backward ? a->dinitial : nullptr};
  for (const void* p : bases)
    if (!aligned(p, 16)) return false;
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
  p.vec = wide(a, true) ? 16 / size_of(a->type) : 1;
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
      const int64_t lanes = a->channels / (w ? 16 / sizeof(T) : 1);
      const int64_t span = a->time ? span_for(a->batch, a->time, lanes, 131072) : 1, stretches = a->time ? ceil_div(a->time, span) : 1;
      const int64_t blocks = ceil_div(a->batch * stretches * lanes, 256);
      if (blocks > 0x7fffffff) return fail(PPN_E_INVALID, "convolution: too many elements");
      if (w) conv_forward<T, K, 16 / sizeof(T)><<<dim3(blocks), dim3(256), 0, (hipStream_t)stream>>>(*a, span, stretches);
      else conv_forward<T, K, 1><<<dim3(blocks), dim3(256), 0, (hipStream_t)stream>>>(*a, span, stretches);
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
  if (p.shares > 65535) return fail(PPN_E_INVALID, "ppn_conv_backward: too many shares");
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return by_taps(a->taps, [&](auto k) {
      constexpr int K = decltype(k)::value;
      const dim3 grid(p.slabs, p.shares);
      if (p.vec > 1) conv_backward<T, K, 16 / sizeof(T)><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a, p.span, p.stretches, (float*)a->workspace);
      else conv_backward<T, K, 1><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a, p.span, p.stretches, (float*)a->workspace);
      conv_reduce<<<dim3(ceil_div((K + 1) * a->channels, 32)), dim3(256), 0, (hipStream_t)stream>>>((const float*)a->workspace, p.shares, a->channels, K,
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
  if (a->rows == 0) return PPN_OK;
  if (!a->x || !a->weight || !a->y || (!a->state && a->environments)) return fail(PPN_E_INVALID, "ppn_conv_step: x, weight, state and y are needed");
  const int64_t vec = 16 / size_of(a->type);
  const bool w = a->channels % vec == 0 && a->x_row % vec == 0 && a->y_row % vec == 0 && aligned(a->x, 16) && aligned(a->y, 16) && aligned(a->state, 16);
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return by_taps(a->taps, [&](auto k) {
      constexpr int K = decltype(k)::value;
      const dim3 grid(a->rows, ceil_div(a->channels / (w ? vec : 1), 256));
      if (grid.y > 65535) return fail(PPN_E_INVALID, "ppn_conv_step: too many channels");
      if (w) conv_step<T, K, 16 / sizeof(T)><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a);
      else conv_step<T, K, 1><<<grid, dim3(256), 0, (hipStream_t)stream>>>(*a);
      return launched("ppn_conv_step");
    });
  });
}
