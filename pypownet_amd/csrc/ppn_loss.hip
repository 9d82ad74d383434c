// ppn_loss.hip -- cross entropy over a catalogue of actions, without keeping the logits.
//
//   loss[i] = log sum_v exp(l[i,v]) - l[i,target]      l[i,v] = hidden[i] . weight[v], over the allowed actions
//   dl[i,v] = (exp(l[i,v] - lse[i]) - [v = target]) dloss[i]      dhidden = dl weight      dweight = dl^T hidden
//
// Bound by the matrix units: 2 rows x actions x features operations forward, three times that and the logits once more backward.  One
// matrix product serves all four: C = A B^T with both operands' inner dimension contiguous, 32-bit sums, and an epilogue that differs:
//   logits -> running maximum and sum of exponentials per row and tile (nothing else leaves the chip),
//   logits -> dl of a piece of the catalogue, rounded to the operands' type and laid out both ways (dl and its transpose),
//   dl and dl^T against transposed copies of weight and hidden -> the two gradients.
// The catalogue is taken in pieces, so that dl needs a bounded workspace whatever the catalogue's size: 256 MB and as much for its transpose, or
// 1024 actions' worth where the rows make that more.
//
// 16384 rows, 24129 actions, 512 features in bfloat16 (405 GFLOP a product): the first kind takes 433 us (935 TFLOP/s), the second 737 us (550; it
// writes 1.6 GB, and the transposed copies), the third 900 us for both (900).  A large library product reaches 1250 TFLOP/s; at these shapes it takes 572 us for the logits
// alone, 466 and 325 us for the other two.  4096 rows: 108 us, and 83 of those are the product without its epilogue (10 vector instructions a logit),
// which the other workgroups of a CU cover in part.
//
// Rounding dl to 16 bits (as the operand of a 16-bit product it has to be) is off by at most half a step of each entry, 2^-8 of it for bfloat16
// and 2^-11 for float16, independent from entry to entry; the gradients' own rounding is as large.  float16's range would lose small
// probabilities, so dl is scaled by a power of two that brings the largest |dloss| to 2^14, and the scale is taken out at the end.
#include "ppn_policy.h"

#include <float.h>

namespace ppn_policy {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// 16 bytes of each operand (of a lane) into a 16 x 16 tile of sums: inner positions (lane / 16) * 16 bytes ..
__device__ inline void multiply(f32x4& c, u32x4 a, u32x4 b, __bf16) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ inline void multiply(f32x4& c, u32x4 a, u32x4 b, _Float16) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ inline void multiply(f32x4& c, u32x4 a, u32x4 b, float) {
  const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
}

// Operands of one product: C[m, n] = sum_k A[m, k] B[n, k]; rows and the inner dimension in whole 16 bytes.
struct Operands {
  const void* A; int64_t lda, M;
  const void* B; int64_t ldb, N;
  int64_t K;
};

struct StatsArgs { const int32_t* allowed; int64_t allowed_row; float2* partial; int64_t columns; };
struct GradArgs {
  const int32_t* allowed; int64_t allowed_row; const int64_t* target; const float* lse; const float* loss; const float* dloss; const float* scale;
  void* dl; int64_t dl_row; void* dlt; int64_t dlt_row; int64_t first, rows_padded, cols_padded;
};
// A product of the backward pass: shares of the inner dimension, `share` long, by tiles; 32-bit sums of share k to sums + k M N (on top of what is
// there with add), or, with one share and nothing to add to, the result itself to out.
struct SumJob { Operands o; float* sums; void* out; int64_t share; unsigned tiles_m, tiles_n, blocks; bool add; };

__device__ const u32x4 zeros = {0, 0, 0, 0};

constexpr int LINE = 128;         // bytes of the inner dimension per stage: a cache line, so that none is brought twice

// Tile of 16 MI WM x 16 NI WN by WM x WN waves of 16 MI x 16 NI.  Both operands' lines go from memory straight into LDS, a stage of one line a row
// at a time.  A stage's fragments are all read into registers, so that the next stage's lines can come in its place while the matrix units work;
// what is waited for in between (the lines' way, the reads), and the epilogue, is covered by the other workgroups of the CU: two of 256 x 128,
// three of 128 x 128.  (Two buffers, a stage ahead, leave room for one workgroup of 256 x 256: 129 us against 112 for the logits of 4096 x 24129
// x 512, whose epilogue then stands alone, and 343 against 313 for the gradients' products of 16384 x 8192 x 512.)  A line's eight 16-byte parts
// are stored with part ^ (row % 8), so that the rows a fragment read touches fall into different banks; the transfer writes 64 lanes' 16 bytes in
// a row (8 lines), so the exchange is made in the addresses it reads.
template <typename T, int MI, int NI, int WM, int WN> struct Product {
  static constexpr int BM = 16 * MI * WM, BN = 16 * NI * WN, THREADS = 64 * WM * WN;
  static constexpr int OF_A = BM / 8 / (WM * WN), OF_B = BN / 8 / (WM * WN), LOADS = OF_A + OF_B;      // a wave's transfers of 8 lines
  static constexpr int LDS_BYTES = (BM + BN) * LINE;
  static_assert(OF_A * 8 * WM * WN == BM && OF_B * 8 * WM * WN == BN, "the lines are shared out evenly");

  f32x4 c[MI][NI];
  int wave_m, wave_n, lane;

  __device__ static int spot(int row, int part) { return row * LINE + ((part ^ (row & 7)) << 4); }

  // 8 lines into LDS at byte `to`.  The transfer is counted by the wave's vector memory counter and nothing else waits for it: see run().  A scalar
  // write of M0 (where the lines go) needs one wait state before the load that reads it; the compiler does not look into assembly for that.
  // (__builtin_amdgcn_global_load_lds would bring it along, but makes branches of the choice of `zeros` and 64-bit vector additions of the addresses.)
  __device__ static void transfer(unsigned to, const char* base, unsigned offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory", "m0");
  }

  // The same with an address a lane, for the last stage where it is not a whole line: what is past its end is read from `zeros`.
  __device__ static void transfer(unsigned to, const char* address) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(address) : "memory", "m0");
  }

  // The same for all lanes of the wave, and in scalar registers; with the five wait states between a vector instruction's write of a scalar register
  // and a memory operation (in the assembly above) that reads it.
  __device__ static const char* scalar(const char* p) {
    const uint64_t v = (uint64_t)p;
    uint64_t r = (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)v);
    asm volatile("s_nop 4" : "+s"(r));
    return (const char*)r;
  }

  __device__ void run(const Operands& o, char* lds, int64_t m0, int64_t n0, int64_t k0, int64_t k1) {
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    lane = tid & 63;
    wave_m = wave / WN * (16 * MI), wave_n = wave % WN * (16 * NI);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) c[i][j] = f32x4{0, 0, 0, 0};
    // this wave's lines: 8 OF_A neighbouring ones of A, 8 OF_B of B; lines past the last one read the last one again
    const int row = lane >> 3, swap = ((lane & 7) ^ row) << 4;
    const unsigned start = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    const unsigned to_a = __builtin_amdgcn_readfirstlane(start + wave * (OF_A * 8 * LINE)), to_b = __builtin_amdgcn_readfirstlane(start + (BM + wave * (OF_B * 8)) * LINE);
    const int64_t first_a = m0 + wave * (OF_A * 8), first_b = n0 + wave * (OF_B * 8);
    const int64_t top_a = first_a < o.M ? first_a : o.M - 1, top_b = first_b < o.N ? first_b : o.N - 1;
    const int spare_a = (int)(o.M - 1 - top_a < 8 * OF_A ? o.M - 1 - top_a : 8 * OF_A), spare_b = (int)(o.N - 1 - top_b < 8 * OF_B ? o.N - 1 - top_b : 8 * OF_B);
    const char* base_a = scalar((const char*)o.A + (top_a * o.lda + k0) * (int64_t)sizeof(T));
    const char* base_b = scalar((const char*)o.B + (top_b * o.ldb + k0) * (int64_t)sizeof(T));
    const unsigned ld_a = (unsigned)(o.lda * sizeof(T)), ld_b = (unsigned)(o.ldb * sizeof(T)), mine_a = row * ld_a + swap, mine_b = row * ld_b + swap;
    const bool whole = spare_a >= 8 * OF_A - 1 && spare_b >= 8 * OF_B - 1;
    const int bytes = (int)((k1 - k0) * (int64_t)sizeof(T)), stages = (bytes + LINE - 1) / LINE;
    auto fetch = [&](int stage) {
      const int left_over = bytes - stage * LINE;
      if (whole && left_over >= LINE) {
#pragma unroll
        for (int i = 0; i < OF_A; ++i) transfer(to_a + i * 8 * LINE, base_a + (uint64_t)i * 8 * ld_a, mine_a);
#pragma unroll
        for (int i = 0; i < OF_B; ++i) transfer(to_b + i * 8 * LINE, base_b + (uint64_t)i * 8 * ld_b, mine_b);
      } else {
        const bool in = swap < left_over;
        int here = row;
        asm volatile("" : "+v"(here));      // (the addresses are made here: kept over the loop they do not fit the registers)
#pragma unroll
        for (int i = 0; i < OF_A; ++i) transfer(to_a + i * 8 * LINE, in ? base_a + (unsigned)min(8 * i + here, spare_a) * ld_a + swap : (const char*)&zeros);
#pragma unroll
        for (int i = 0; i < OF_B; ++i) transfer(to_b + i * 8 * LINE, in ? base_b + (unsigned)min(8 * i + here, spare_b) * ld_b + swap : (const char*)&zeros);
      }
      base_a += LINE, base_b += LINE;
    };
    struct Fragments { u32x4 a[MI], b[NI]; };
    int at_a[2], at_b[2];      // where this lane's fragments begin, by half; rows 16 apart have the same row % 8
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      at_a[h] = spot(wave_m + (lane & 15), 4 * h + (lane >> 4));
      at_b[h] = spot(BM + wave_n + (lane & 15), 4 * h + (lane >> 4));
    }
    auto read = [&](Fragments& f, int h) {
#pragma unroll
      for (int j = 0; j < NI; ++j) f.b[j] = *(const u32x4*)(lds + at_b[h] + j * 16 * LINE);
#pragma unroll
      for (int i = 0; i < MI; ++i) f.a[i] = *(const u32x4*)(lds + at_a[h] + i * 16 * LINE);
    };
    auto multiply_all = [&](const Fragments& f) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) multiply(c[i][j], f.a[i], f.b[j], T());
    };
    fetch(0);
    for (int s = 0; s < stages; ++s) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // the stage's lines are in, every wave's
      Fragments even, odd;
      read(even, 0);
      read(odd, 1);
      // Every wave has the stage's fragments in registers: the next stage's lines may come in their place.
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (s + 1 < stages) fetch(s + 1);
      multiply_all(even);
      multiply_all(odd);
    }
  }
  // Sum (i, j, r) of this lane: row wave_m + 16 i + 4 (lane / 16) + r, column wave_n + 16 j + lane % 16 of the tile.
  __device__ int row_of(int i, int r) const { return wave_m + i * 16 + (lane >> 4) * 4 + r; }
  __device__ int col_of(int j) const { return wave_n + j * 16 + (lane & 15); }
};

// Which tile a workgroup takes.  Workgroups are handed to the eight dies in turn, each with its own 4 MB of L2: neighbours in the list below go to
// one die, and the list goes through eight tiles of rows (2 MB at 256 rows of 512 16-bit features) for every tile of columns, so that a die
// keeps its rows and reads the columns once.  In the order of the rows alone 16384 x 24129 x 512 read 1.8 GB instead of 0.2.
__device__ inline void tile_of(unsigned id, unsigned tiles_m, unsigned tiles_n, unsigned* m, unsigned* n) {
  const unsigned count = tiles_m * tiles_n, per = count / 8, whole = per * 8, tile = id < whole ? (id % 8) * per + id / 8 : id;
  const unsigned group = tile / (8 * tiles_n), first = group * 8, rows = tiles_m - first < 8 ? tiles_m - first : 8, rest = tile - first * tiles_n;
  *m = first + rest % rows;
  *n = rest / rows;
}

// The 16 lanes of a row of lanes hold one row's columns: their maximum, or sum, for four rows at once.  Written out because the compiler puts a
// quieting instruction and a separate move in front of every maximum.  A lane exchange may follow the write of what it reads by two other
// instructions: two idle ones in front, the other three rows' in between.
#define PPN_OVER_16(OP)                                                                                                                       \
  "s_nop 1\n"                                                                                                                                 \
  OP " %0, %0, %0 row_ror:8 row_mask:0xf bank_mask:0xf\n" OP " %1, %1, %1 row_ror:8 row_mask:0xf bank_mask:0xf\n"                             \
  OP " %2, %2, %2 row_ror:8 row_mask:0xf bank_mask:0xf\n" OP " %3, %3, %3 row_ror:8 row_mask:0xf bank_mask:0xf\n"                             \
  OP " %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n" OP " %1, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xf\n"                 \
  OP " %2, %2, %2 row_half_mirror row_mask:0xf bank_mask:0xf\n" OP " %3, %3, %3 row_half_mirror row_mask:0xf bank_mask:0xf\n"                 \
  OP " %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n" OP " %1, %1, %1 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"         \
  OP " %2, %2, %2 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n" OP " %3, %3, %3 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"         \
  OP " %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n" OP " %1, %1, %1 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"         \
  OP " %2, %2, %2 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n" OP " %3, %3, %3 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
__device__ inline void max_over_16(float (&v)[4]) { asm volatile(PPN_OVER_16("v_max_f32_dpp") : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3])); }
__device__ inline void sum_over_16(float (&v)[4]) { asm volatile(PPN_OVER_16("v_add_f32_dpp") : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3])); }
#undef PPN_OVER_16
// Plain maxima, the same way (arguments are results of ordinary instructions, never of a matrix instruction: those need waits of their own).
__device__ inline float most(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ inline float most(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// a where the bit of the word is set, else b: two instructions, and nothing of a is looked at where it is not.
__device__ inline float chosen(unsigned word, int bit, float a, int b) {
  const int yes = __builtin_amdgcn_sbfe((int)word, bit, 1);
  return __builtin_bit_cast(float, (yes & __builtin_bit_cast(int, a)) | (~yes & b));
}

// The bits of BN columns from n0 (of N, whose word 0 is `word` words into a row of allowed) that row `row` may count: none past the last
// column.  Called before the product, so that the loads' way is covered by it; read after it.
template <int BN> __device__ inline void stage_mask(unsigned (*mask)[BN / 32], int at, const int32_t* allowed, int64_t allowed_row, int64_t row, int64_t word, int64_t n0, int64_t N,
                                                    bool live) {
#pragma unroll
  for (int w = 0; w < BN / 32; ++w) {
    const int64_t left = N - n0 - 32 * w;
    unsigned bits = left >= 32 ? ~0u : left > 0 ? (1u << left) - 1 : 0;
    if (!live) bits = 0;
    if (allowed && bits) bits &= (unsigned)allowed[row * allowed_row + word + n0 / 32 + w];
    mask[at][w] = bits;
  }
}

// Forward: of every row and every 16 NI columns the maximum and the sum of exp(l - maximum), [columns / 16 NI x rows].  Logarithms to base 2.
template <typename T, int MI, int NI, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) loss_stats(Operands o, StatsArgs s, unsigned tiles_m, unsigned tiles_n) {
  typedef Product<T, MI, NI, WM, WN> P;
  __shared__ __align__(16) char lds[P::LDS_BYTES];
  __shared__ __align__(16) unsigned mask[P::BM][P::BN / 32];
  unsigned tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, &tm, &tn);
  const int64_t m0 = (int64_t)tm * P::BM, n0 = (int64_t)tn * P::BN;
  for (int r = threadIdx.x; r < P::BM; r += P::THREADS)
    stage_mask<P::BN>(mask, r, s.allowed, s.allowed_row, m0 + r < o.M ? m0 + r : o.M - 1, 0, n0, o.N, true);
  P p;
  p.run(o, lds, m0, n0, 0, o.K);
  const int column = p.lane & 15, next = column + 16;      // this lane's bit in a word's halves
  float2* out = s.partial + (n0 + p.wave_n) / (16 * NI) * o.M + m0;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    float l[4][NI], top[4], sum[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const unsigned* word = mask[p.row_of(i, r)] + p.wave_n / 32;
#pragma unroll
      for (int j = 0; j < NI; ++j) l[r][j] = chosen(word[j / 2], j & 1 ? next : column, p.c[i][j][r], (int)0xff800000);      // -infinity
      if constexpr (NI == 8) top[r] = most(most(most(l[r][0], l[r][1], l[r][2]), l[r][3], l[r][4]), most(l[r][5], l[r][6], l[r][7]));
      else if constexpr (NI == 4) top[r] = most(most(l[r][0], l[r][1], l[r][2]), l[r][3]);
      else top[r] = most(l[r][0], l[r][1]);
    }
    max_over_16(top);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      top[r] *= LOG2E;
      const float ref = top[r] == -INFINITY ? 0.0f : top[r];
      sum[r] = 0.0f;
#pragma unroll
      for (int j = 0; j < NI; ++j) sum[r] += __builtin_amdgcn_exp2f(l[r][j] * LOG2E - ref);
    }
    sum_over_16(sum);
    // lanes 0..3 of each 16 have a row to write
    float t = column & 2 ? (column & 1 ? top[3] : top[2]) : (column & 1 ? top[1] : top[0]);
    const float u = column & 2 ? (column & 1 ? sum[3] : sum[2]) : (column & 1 ? sum[1] : sum[0]);
    const int row = p.row_of(i, column);
    if (column < 4 && m0 + row < o.M) {
      if (t == -INFINITY) {      // nothing allowed here, or allowed logits of minus infinity: the latter leave the lowest number
        unsigned any = 0;
#pragma unroll
        for (int j = 0; j < NI; j += 2) any |= mask[row][p.wave_n / 32 + j / 2];
        if (any) t = -FLT_MAX;
      }
      out[row] = make_float2(t, u);
    }
  }
}

// Sixteen rows a workgroup: joins the tiles' maxima and sums, 16 lanes a row, and takes the target's logit as a product of its own, a wave a row (four
// rows' worth of loads at a time).
template <typename T>
__global__ void __launch_bounds__(256) loss_join(ppn_loss_args a, const float2* partial, int64_t columns) {
  __shared__ float tops[16][17], sums[16][17], wanted[16];
  const int64_t first = (int64_t)blockIdx.x * 16;
  const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
  {
    const int64_t row = first + (threadIdx.x & 15) < a.rows ? first + (threadIdx.x & 15) : a.rows - 1;
    float top = -INFINITY, sum = 0.0f;
    // (a tile without an allowed action has the sum 0 and the maximum -infinity; one whose allowed logits are all -infinity the sum 0 and the lowest
    // number; one with a NaN has the sum NaN whatever its maximum)
    constexpr int AHEAD = 4;
    for (int64_t c = threadIdx.x / 16; c < columns; c += 16 * AHEAD) {
      float2 v[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int64_t at = c + 16 * k;
        v[k] = partial[(at < columns ? at : c) * a.rows + row];
        if (at >= columns) v[k] = make_float2(-INFINITY, 0.0f);
      }
      float high = top;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) high = fmaxf(high, v[k].x);
      const float ref = high == -INFINITY ? 0.0f : high;
      sum *= __builtin_amdgcn_exp2f(top - ref);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) sum += v[k].y * __builtin_amdgcn_exp2f(v[k].x - ref);
      top = high;
    }
    tops[threadIdx.x & 15][threadIdx.x / 16] = top;
    sums[threadIdx.x & 15][threadIdx.x / 16] = sum;
  }
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const T* h[4];
  const T* w[4];
  bool inside[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t row = first + wave * 4 + k < a.rows ? first + wave * 4 + k : a.rows - 1, at = a.target[row];
    inside[k] = at >= 0 && at < a.actions;
    h[k] = (const T*)a.hidden + row * a.hidden_row;
    w[k] = (const T*)a.weight + (inside[k] ? at : 0) * a.weight_row;
  }
  for (int64_t f = lane; f < a.features; f += 64)
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] += to_float(h[k][f]) * to_float(w[k][f]);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    for (int d = 32; d; d >>= 1) s[k] += __shfl_xor(s[k], d);
    if (lane == 0) wanted[wave * 4 + k] = s[k];
  }
  __syncthreads();
  if (threadIdx.x >= 16 || first + threadIdx.x >= a.rows) return;
  const int64_t row = first + threadIdx.x, at = a.target[row];
  float top = -INFINITY, sum = 0.0f;
  for (int k = 0; k < 16; ++k) top = fmaxf(top, tops[threadIdx.x][k]);
  const float ref = top == -INFINITY ? 0.0f : top;
  for (int k = 0; k < 16; ++k) sum += sums[threadIdx.x][k] * __builtin_amdgcn_exp2f(tops[threadIdx.x][k] - ref);
  const bool nothing = top == -INFINITY && sum == 0.0f, known = at >= 0 && at < a.actions;
  const float whole = 0.693147180559945309f * (top + __builtin_amdgcn_logf(sum));
  float loss = 0.0f, lse = INFINITY;
  if (at != a.ignore_index && !nothing) {
    const bool legal = known && (!a.allowed || ((a.allowed[row * a.allowed_row + (at >> 5)] >> (at & 31)) & 1));
    const bool undefined = !known || fabsf(whole) == INFINITY;      // (a logit of infinity, or none above -infinity: there are no shares)
    loss = !known ? NAN : !legal ? INFINITY : undefined ? NAN : whole - wanted[threadIdx.x];
    lse = undefined ? NAN : whole;
  }
  a.loss[row] = loss;
  a.lse[row] = lse;
}

// float16: scale[0], the power of two dl is multiplied by (it brings the largest |dloss| to 2^14), and scale[1] = 1 / scale[0].
__global__ void __launch_bounds__(1024) loss_scale(const float* dloss, const float* lse, int64_t rows, float* scale) {
  __shared__ float tops[1024];
  float top = 0.0f;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    const float g = fabsf(dloss[i]);
    if (lse[i] != INFINITY && g < INFINITY && g > top) top = g;
  }
  tops[threadIdx.x] = top;
  __syncthreads();
  for (int half = 512; half; half >>= 1) {
    if (threadIdx.x < half) tops[threadIdx.x] = fmaxf(tops[threadIdx.x], tops[threadIdx.x + half]);
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    top = tops[0];
    int e = 0;
    if (top > 0.0f) frexpf(top, &e);
    e = e < -100 ? -100 : e > 100 ? 100 : e;
    scale[0] = top > 0.0f ? ldexpf(1.0f, 14 - e) : 1.0f;
    scale[1] = top > 0.0f ? ldexpf(1.0f, e - 14) : 1.0f;
  }
}

// The transposed copies of hidden and weight, [cols x rows_padded] with zeros in the padding, for the second products: 64 x 64 tiles through LDS, `across`
// of them along the rows, by workgroups in the launch that makes dl (of 999 x 12099 x 392: 31 us together, 25 and 13 apart).  A row of hidden without a gradient (lse +infinity) becomes zeros:
// whatever stands in it, its product with dl's zeros is zero.
struct TransposeJob { const void* in; int64_t in_row, rows, cols; void* out; int64_t rows_padded; const float* lse; unsigned across, blocks; };
template <typename T> constexpr int TRANSPOSE_BYTES = 64 * (64 + 4 / sizeof(T)) * sizeof(T);
template <typename T> __device__ inline void transpose(const TransposeJob& job, unsigned id, char* lds) {
  typedef T Line[64 + 4 / sizeof(T)];
  Line* tile = (Line*)lds;
  const int64_t r0 = (int64_t)(id % job.across) * 64, c0 = (int64_t)(id / job.across) * 64;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const T* in = (const T*)job.in;
  T part[16];
  float lse[16];
  const int64_t column = c0 + x < job.cols ? c0 + x : job.cols - 1;
  const float* marks = job.lse ? job.lse : (const float*)job.out;      // (read in its place and not looked at)
  const int64_t mark_step = job.lse ? 1 : 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {      // (loads without a branch, all in flight)
    const int64_t r = r0 + y + 4 * i, row = r < job.rows ? r : job.rows - 1;
    part[i] = in[row * job.in_row + column];
    lse[i] = marks[row * mark_step];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const bool out = r0 + y + 4 * i >= job.rows || c0 + x >= job.cols || (job.lse && lse[i] == INFINITY);
    tile[y + 4 * i][x] = out ? (T)0.0f : part[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 64; i += 4) {
    const int64_t c = c0 + y + i, r = r0 + x;
    if (c < job.cols && r < job.rows_padded) ((T*)job.out)[c * job.rows_padded + r] = tile[x][y + i];
  }
}

// Two rows' (of a lane's column) values as one word, and the exchange that turns four rows of one column into two rows of two columns: lanes of
// even columns keep the first two rows, those of odd ones the last two.
__device__ inline unsigned pair(__bf16 a, __bf16 b) { return (unsigned)__builtin_bit_cast(unsigned short, a) | (unsigned)__builtin_bit_cast(unsigned short, b) << 16; }
__device__ inline unsigned pair(_Float16 a, _Float16 b) { return (unsigned)__builtin_bit_cast(unsigned short, a) | (unsigned)__builtin_bit_cast(unsigned short, b) << 16; }
__device__ inline unsigned from_neighbour(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true); }      // quad_perm 1,0,3,2

// Backward, first product: dl of the columns first .. first + N of the catalogue, [rows x cols_padded] and [N x rows_padded], zeros in the padding.
// The target's own entry, (e^-loss - 1) dloss, is written over its tile's value at the end.
template <typename T, int MI, int NI, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) loss_grad(Operands o, GradArgs g, unsigned tiles_m, unsigned tiles_n, TransposeJob one, TransposeJob two) {
  typedef Product<T, MI, NI, WM, WN> P;
  struct Row { float lse2, up; };
  static_assert(P::THREADS == 256, "transpose()");
  constexpr int OUT = sizeof(T) == 2 ? P::BM * P::BN * 2 : TRANSPOSE_BYTES<T>;
  __shared__ __align__(16) char lds[P::LDS_BYTES > OUT ? P::LDS_BYTES : OUT];
  static_assert(sizeof lds >= TRANSPOSE_BYTES<T>, "transpose()");
  __shared__ __align__(16) unsigned mask[P::BM][P::BN / 32];
  __shared__ __align__(16) Row rows[P::BM];
  const unsigned tiles = tiles_m * tiles_n;
  if (blockIdx.x >= tiles) {
    const unsigned id = blockIdx.x - tiles;
    if (id < one.blocks) transpose<T>(one, id, lds);
    else transpose<T>(two, id - one.blocks, lds);
    return;
  }
  unsigned tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, &tm, &tn);
  const int64_t m0 = (int64_t)tm * P::BM, n0 = (int64_t)tn * P::BN;
  for (int r = threadIdx.x; r < P::BM; r += P::THREADS) {
    const int64_t row = m0 + r < o.M ? m0 + r : o.M - 1;
    const float lse = g.lse[row];
    const bool live = m0 + r < o.M && lse != INFINITY;                   // a row without a gradient, or past the last one: zeros
    stage_mask<P::BN>(mask, r, g.allowed, g.allowed_row, row, g.first / 32, n0, o.N, live);
    rows[r] = Row{lse * LOG2E, live ? g.dloss[row] * (g.scale ? g.scale[0] : 1.0f) : 0.0f};
  }
  P p;
  p.run(o, lds, m0, n0, 0, o.K);
  const int column = p.lane & 15;
  const unsigned dl_row = (unsigned)g.dl_row * sizeof(T), dlt_row = (unsigned)g.dlt_row * sizeof(T);
  char* dl = (char*)g.dl + (m0 * g.dl_row + n0) * (int64_t)sizeof(T);
  char* dlt = (char*)g.dlt + (n0 * g.dlt_row + m0) * (int64_t)sizeof(T);
  auto entry = [&](int i, int j, int r) {
    const Row q = rows[p.row_of(i, r)];
    const float v = __builtin_amdgcn_exp2f(p.c[i][j][r] * LOG2E - q.lse2) * q.up;
    return (T)chosen(mask[p.row_of(i, r)][p.wave_n / 32 + j / 2], column + (j & 1 ? 16 : 0), v, 0);
  };
  // The entry of a row's target, exact where the probability is near one: (column of the tile, or -1; value).
  struct Hit { int at; T v; };
  auto target_of = [&](int r) {
    Hit hit = {-1, (T)0.0f};
    if (m0 + r >= o.M || g.lse[m0 + r] == INFINITY) return hit;
    const int64_t target = g.target[m0 + r] - g.first - n0;
    if (target < 0 || target >= P::BN || n0 + target >= o.N || !((mask[r][target / 32] >> (target & 31)) & 1)) return hit;
    const float loss = g.loss[m0 + r];
    hit.at = (int)target;
    hit.v = (T)((loss != loss ? loss : expm1f(-loss)) * rows[r].up);
    return hit;
  };
  if constexpr (sizeof(T) == 2) {
    // The tile goes out through LDS, where the operands were, once by rows and once by columns, 16 bytes a lane and whole lines: straight from the
    // registers it would be runs of 32 bytes (312 us against 260 for a piece of 16384 x 8192).  A line's 16-byte parts are exchanged as in the
    // product, so that the lanes of a write fall into different banks.
    constexpr int ROW = P::BN * 2, COL = P::BM * 2, CHUNKS = P::BM * P::BN / 8, EACH = CHUNKS / P::THREADS, BATCH = EACH < 4 ? EACH : 4;
    static_assert(P::BM <= P::THREADS && EACH % BATCH == 0, "the tile fits where the operands were");
    auto in_row = [&](int row, int bytes) { return row * ROW + ((((bytes >> 4) ^ (row >> 1 & 7)) << 4) | (bytes & 15)); };
    auto in_col = [&](int col, int bytes) { return col * COL + ((((bytes >> 4) ^ (col & 7)) << 4) | (bytes & 15)); };
    unsigned q[MI][NI][2];
    Hit hit = {-1, (T)0.0f};
    if (threadIdx.x < P::BM) hit = target_of(threadIdx.x);
    __syncthreads();      // (the last fragments have been read)
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const unsigned a = pair(entry(i, j, 0), entry(i, j, 1)), b = pair(entry(i, j, 2), entry(i, j, 3));
        q[i][j][0] = a, q[i][j][1] = b;
        const bool odd = column & 1;
        const unsigned keep = odd ? b : a, got = from_neighbour(odd ? a : b);
        const unsigned left = odd ? got : keep, right = odd ? keep : got;      // columns col & ~1 and the next, two rows each
        const unsigned lower = __builtin_amdgcn_perm(right, left, 0x05040100), upper = __builtin_amdgcn_perm(right, left, 0x07060302);
        const int row = p.row_of(i, 0) + (odd ? 2 : 0), at = (p.col_of(j) & ~1) * 2;
        *(unsigned*)(lds + in_row(row, at)) = lower;
        *(unsigned*)(lds + in_row(row + 1, at)) = upper;
      }
    __syncthreads();
    if (hit.at >= 0) *(T*)(lds + in_row(threadIdx.x, hit.at * 2)) = hit.v;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EACH; k += BATCH) {
      u32x4 part[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int id = threadIdx.x + (k + u) * P::THREADS;
        part[u] = *(const u32x4*)(lds + in_row(id / (ROW / 16), id % (ROW / 16) * 16));
      }
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int id = threadIdx.x + (k + u) * P::THREADS, row = id / (ROW / 16), at = id % (ROW / 16) * 16;
        if (m0 + row < o.M && n0 + at / 2 < g.cols_padded) *(u32x4*)(dl + (row * dl_row + at)) = part[u];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) *(uint2*)(lds + in_col(p.col_of(j), p.row_of(i, 0) * 2)) = uint2{q[i][j][0], q[i][j][1]};
    __syncthreads();
    if (hit.at >= 0) *(T*)(lds + in_col(hit.at, threadIdx.x * 2)) = hit.v;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EACH; k += BATCH) {
      u32x4 part[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int id = threadIdx.x + (k + u) * P::THREADS;
        part[u] = *(const u32x4*)(lds + in_col(id / (COL / 16), id % (COL / 16) * 16));
      }
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int id = threadIdx.x + (k + u) * P::THREADS, col = id / (COL / 16), at = id % (COL / 16) * 16;
        if (n0 + col < o.N && m0 + at / 2 < g.rows_padded) *(u32x4*)(dlt + (col * dlt_row + at)) = part[u];
      }
    }
  } else {
    const bool whole = m0 + P::BM <= o.M && n0 + P::BN <= o.N;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int row0 = p.row_of(i, 0), col = p.col_of(j);
        const f32x4 f = {entry(i, j, 0), entry(i, j, 1), entry(i, j, 2), entry(i, j, 3)};
        if (whole || (n0 + col < o.N && m0 + row0 < g.rows_padded))      // rows_padded is a multiple of 16: the four rows are in or out together
          *(f32x4*)(dlt + (col * dlt_row + row0 * 4u)) = f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (whole || (m0 + row0 + r < o.M && n0 + col < g.cols_padded)) *(float*)(dl + ((row0 + r) * dl_row + col * 4u)) = f[r];
      }
    // the targets' entries, behind the tile's own stores
    __threadfence_block();
    __syncthreads();
    for (int r = threadIdx.x; r < P::BM; r += P::THREADS) {
      const Hit hit = target_of(r);
      if (hit.at < 0) continue;
      *(float*)(dl + (r * dl_row + hit.at * 4u)) = hit.v;
      *(float*)(dlt + (hit.at * dlt_row + r * 4u)) = hit.v;
    }
  }
}

// Backward, second products: dhidden's and dweight's at once, so that the one fills the CUs the other leaves.
template <typename T, int MI, int NI, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) loss_sums(SumJob one, SumJob two, const float* scale) {
  typedef Product<T, MI, NI, WM, WN> P;
  __shared__ __align__(16) char lds[P::LDS_BYTES];
  const bool second = blockIdx.x >= one.blocks;
  const SumJob job = second ? two : one;
  const Operands& o = job.o;
  const unsigned id = blockIdx.x - (second ? one.blocks : 0), tiles = job.tiles_m * job.tiles_n, k = id / tiles;
  unsigned tm, tn;
  tile_of(id - k * tiles, job.tiles_m, job.tiles_n, &tm, &tn);
  const int64_t m0 = (int64_t)tm * P::BM, n0 = (int64_t)tn * P::BN, k0 = k * job.share, k1 = k0 + job.share < o.K ? k0 + job.share : o.K;
  P p;
  p.run(o, lds, m0, n0, k0, k1);
  const unsigned ld = (unsigned)o.N;
  const bool whole = m0 + P::BM <= o.M && n0 + P::BN <= o.N;
  if (job.out) {
    T* out = (T*)job.out + m0 * o.N + n0;
    const float unscale = scale ? scale[1] : 1.0f;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < NI; ++j)
          if (whole || (m0 + p.row_of(i, r) < o.M && n0 + p.col_of(j) < o.N)) out[p.row_of(i, r) * ld + p.col_of(j)] = (T)(p.c[i][j][r] * unscale);
    return;
  }
  float* sums = job.sums + k * o.M * o.N + m0 * o.N + n0;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    float old[4][NI];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        old[r][j] = 0.0f;
        if (job.add && (whole || (m0 + p.row_of(i, r) < o.M && n0 + p.col_of(j) < o.N))) old[r][j] = sums[p.row_of(i, r) * ld + p.col_of(j)];
      }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < NI; ++j)
        if (whole || (m0 + p.row_of(i, r) < o.M && n0 + p.col_of(j) < o.N)) sums[p.row_of(i, r) * ld + p.col_of(j)] = old[r][j] + p.c[i][j][r];
  }
}

// What is left to do with the products' 32-bit sums: two jobs (dhidden, dweight), `count` elements of `slots` slots each.
struct FinishJob { const float* sums; int64_t slots, count; void* out; };
template <typename T>
__global__ void __launch_bounds__(256) loss_finish(FinishJob one, FinishJob two, int64_t blocks_one, const float* scale) {
  const bool second = blockIdx.x >= blocks_one;
  const FinishJob job = second ? two : one;
  const int64_t i = ((int64_t)blockIdx.x - (second ? blocks_one : 0)) * 256 + threadIdx.x;
  if (i >= job.count) return;
  float v = 0.0f;
  for (int64_t s = 0; s < job.slots; ++s) v += job.sums[s * job.count + i];
  ((T*)job.out)[i] = (T)(scale ? v * scale[1] : v);
}

// [rows x cols] with any row stride -> [rows x cols_padded], zeros in the padding.
template <typename T>
__global__ void __launch_bounds__(256) loss_pad(const T* in, int64_t in_row, int64_t rows, int64_t cols, T* out, int64_t cols_padded) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * cols_padded) return;
  const int64_t r = i / cols_padded, c = i - r * cols_padded;
  out[i] = c < cols ? in[r * in_row + c] : (T)0.0f;
}

// ---- plans -------------------------------------------------------------------------------------------------------------------------
int64_t padded(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t part(const ppn_loss_args* a) { return 16 / size_of(a->type); }      // elements of 16 bytes

// Rows that the product reads as they are; others are copied into whole 16 bytes first.
bool in_place(const void* p, int64_t row, int64_t features, int64_t type) {
  return features % (16 / size_of(type)) == 0 && row * size_of(type) % 16 == 0 && row <= (1 << 23) && aligned(p, 16);
}

struct Config { int64_t m, n, columns_per_wave; };
constexpr Config LARGE = {256, 128, 64}, MEDIUM = {128, 128, 128}, SMALL = {64, 64, 32};
// The logits: 128 x 128 tiles where they make one and a half workgroups a CU, else 64 x 64.  At 256 x 128, 128 and 64, in us: 116, 112, 151 for 4096 x
// 24129 x 512; 22, 21, 28 for 999 x 12099 x 392; -, 13, 6 for 256 x 347 x 128 in 32 bits.  The waves are 32 x 128: the epilogue's sums over a
// row's columns cost half of what they do in 64 x 64.
Config config_for(int64_t m, int64_t n) { return ceil_div(m, 128) * ceil_div(n, 128) >= 384 ? MEDIUM : SMALL; }
// f(fragments of a wave across the rows, across the columns, waves across the rows, across the columns)
template <int MI, int NI, int WM, int WN> struct Shape { static constexpr int mi = MI, ni = NI, wm = WM, wn = WN; };
template <typename F> void by_tile(const Config& c, F f) {
  if (c.m == 128) f(Shape<2, 8, 4, 1>());
  else f(Shape<2, 2, 2, 2>());
}
template <typename F> void by_large_tile(const Config& c, F f) {
  if (c.m == 256) f(Shape<8, 4, 2, 2>());
  else by_tile(c, f);
}

struct Layout { int64_t bytes = 0; int64_t take(int64_t n) { int64_t at = bytes; bytes += padded(n, 256); return at; } };

struct ForwardPlan { Config config; int64_t columns, features_padded, hidden, weight, partial, bytes; };
ForwardPlan plan_forward(const ppn_loss_args* a) {
  ForwardPlan p;
  Layout l;
  const int64_t size = size_of(a->type);
  p.features_padded = padded(a->features, part(a));
  p.config = config_for(a->rows, a->actions);
  p.columns = padded(a->actions, p.config.n) / p.config.columns_per_wave;
  p.hidden = in_place(a->hidden, a->hidden_row, a->features, a->type) ? -1 : l.take(a->rows * p.features_padded * size);
  p.weight = in_place(a->weight, a->weight_row, a->features, a->type) ? -1 : l.take(a->actions * p.features_padded * size);
  p.partial = l.take(a->rows * p.columns * 8);
  p.bytes = l.bytes;
  return p;
}

struct BackwardPlan {
  int64_t features_padded, rows_padded, actions_padded, piece, hidden, weight, hidden_t, weight_t, dl, dlt, scale, dh, dw, bytes;
  Config grad, sums;
  int64_t share, dh_slots, dw_slots;
  bool direct_dh, direct_dw;
};

// (The same whether both gradients are wanted or one: the sizes alone tell how much memory a call needs.)
BackwardPlan plan_backward(const ppn_loss_args* a) {
  BackwardPlan p;
  Layout l;
  const int64_t size = size_of(a->type);
  p.features_padded = padded(a->features, part(a));
  p.rows_padded = padded(a->rows, 64);
  p.actions_padded = padded(a->actions, 64);
  // A piece's dl and its transpose take 256 MB each, or 1024 actions times the rows where that is more (above 131072 rows in 16 bits, 65536 in 32: the
  // rows are not taken in pieces).  The smaller the piece, the shorter the inner dimension of dhidden's product and the fewer tiles
  // of dweight's: 16384 rows of 24129 actions took 3.65, 3.02, 2.71 and 2.44 ms behind the loss at 32, 64, 128 and 256 MB; with both products in a
  // launch 256, 512 and 1024 MB are within 2 % of each other.
  p.piece = padded((int64_t)(256 << 20) / (p.rows_padded * size), 128);
  if (p.piece < 1024) p.piece = 1024;
  if (p.piece > p.actions_padded) p.piece = p.actions_padded;
  // dl: 256 x 128 where two rounds of them fill the chip (16384 x 8192: 255 us, 269 in 128 x 128; 999 x 12099: 27 and 25)
  p.grad = ceil_div(a->rows, 256) * ceil_div(p.piece, 128) >= 1024 ? LARGE : config_for(a->rows, p.piece);
  // The second products: the largest tile with which shares of at least 512 of the inner dimensions make 384 workgroups of the two, then the
  // shortest share with which they are at most 512.  (Where dhidden's tiles alone come near 512 that is the longest inner dimension, and dweight's product
  // stays in one share: right, but on few workgroups.  Training steps of 16384, 20480 and 61440 rows x 24129 x 512 take 2.06, 3.3 and 20 ms.)  At 256 x 128, 128 and 64, in us: 48, 55, 113 for 999 x 12099 x 392; -, 35, 12 for 256 x 347 x
  // 128 in 32 bits.
  for (int i = 0; i < 3; ++i) {
    p.sums = i == 0 ? LARGE : i == 1 ? MEDIUM : SMALL;
    const int64_t across = ceil_div(a->features, p.sums.n), dh = ceil_div(a->rows, p.sums.m) * across, dw = ceil_div(p.piece, p.sums.m) * across;
    auto blocks = [&](int64_t share) { return dh * ceil_div(p.piece, share) + dw * ceil_div(p.rows_padded, share); };
    if (i < 2 && blocks(512) < 384) continue;
    p.share = 512;
    const int64_t longest = p.piece > p.rows_padded ? p.piece : p.rows_padded;
    while (p.share < longest && blocks(p.share) > 512) p.share += 128;
    break;
  }
  p.dh_slots = ceil_div(p.piece, p.share), p.dw_slots = ceil_div(p.rows_padded, p.share);
  p.direct_dh = p.dh_slots == 1 && p.piece >= a->actions, p.direct_dw = p.dw_slots == 1;
  p.hidden = in_place(a->hidden, a->hidden_row, a->features, a->type) ? -1 : l.take(a->rows * p.features_padded * size);
  p.weight = in_place(a->weight, a->weight_row, a->features, a->type) ? -1 : l.take(a->actions * p.features_padded * size);
  p.hidden_t = l.take(a->features * p.rows_padded * size);
  p.weight_t = l.take(a->features * p.actions_padded * size);
  p.dl = l.take(a->rows * p.piece * size);
  p.dlt = l.take(p.piece * p.rows_padded * size);
  p.scale = l.take(8);
  p.dh = l.take(p.direct_dh ? 0 : p.dh_slots * a->rows * a->features * 4);
  p.dw = l.take(p.direct_dw ? 0 : p.dw_slots * p.piece * a->features * 4);
  p.bytes = l.bytes;
  return p;
}

int check(const ppn_loss_args* a) {
  if (!a || a->struct_bytes != (int64_t)sizeof *a) return fail(PPN_E_INVALID, "ppn_loss_args: struct_bytes does not match this library");
  if (a->type < 0 || a->type > PPN_T_F16) return fail(PPN_E_INVALID, "element type %lld is unknown", (long long)a->type);
  if (a->rows < 0 || a->actions < 1 || a->features < 1) return fail(PPN_E_INVALID, "loss: rows >= 0, actions >= 1 and features >= 1 are needed");
  if (a->rows > (1 << 22) || a->actions > (1 << 23) || a->features > (1 << 20))
    return fail(PPN_E_INVALID, "loss: at most 2^22 rows, 2^23 actions and 2^20 features, got %lld, %lld and %lld", (long long)a->rows, (long long)a->actions, (long long)a->features);
  return PPN_OK;
}

// Rows of allowed lie apart, or are all the same one (stride 0).
bool mask_fits(const ppn_loss_args* a) { return !a->allowed || a->rows <= 1 || a->allowed_row == 0 || a->allowed_row >= ceil_div(a->actions, 32); }

template <typename T> void pad_rows(const void* in, int64_t row, int64_t rows, int64_t cols, void* out, int64_t cols_padded, hipStream_t s) {
  loss_pad<T><<<dim3(ceil_div(rows * cols_padded, 256)), dim3(256), 0, s>>>((const T*)in, row, rows, cols, (T*)out, cols_padded);
}

// Every launch of a call, before the first of them.
template <typename Plan> bool pads_fit(const ppn_loss_args* a, const Plan& p) {
  return (p.hidden < 0 || !too_many(ceil_div(a->rows * p.features_padded, 256), 256)) && (p.weight < 0 || !too_many(ceil_div(a->actions * p.features_padded, 256), 256));
}
bool launches_fit(const ppn_loss_args* a, const ForwardPlan& p) {
  return pads_fit(a, p) && !too_many(ceil_div(a->rows, p.config.m) * ceil_div(a->actions, p.config.n), 256);
}
bool launches_fit(const ppn_loss_args* a, const BackwardPlan& p) {
  const int64_t down = ceil_div(a->features, 64), across = ceil_div(a->features, p.sums.n);
  const int64_t grad = ceil_div(a->rows, p.grad.m) * ceil_div(p.piece, p.grad.n) + (ceil_div(p.rows_padded, 64) + ceil_div(p.actions_padded, 64)) * down;
  const int64_t sums = across * (ceil_div(a->rows, p.sums.m) * p.dh_slots + ceil_div(p.piece, p.sums.m) * p.dw_slots);
  const int64_t finish = ceil_div(a->rows * a->features, 256) + ceil_div(p.piece * a->features, 256);
  return pads_fit(a, p) && !too_many(grad, 256) && !too_many(sums, 256) && !too_many(finish, 256);
}

}  // namespace
}  // namespace ppn_policy

using namespace ppn_policy;

extern "C" int64_t ppn_loss_forward_workspace(const ppn_loss_args* a) {
  if (int rc = check(a)) return rc;
  return plan_forward(a).bytes;
}

extern "C" int ppn_loss_forward(const ppn_loss_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  if (a->rows == 0) return PPN_OK;
  if (!a->hidden || !a->weight || !a->target || !a->loss || !a->lse) return fail(PPN_E_INVALID, "ppn_loss_forward: hidden, weight, target, loss and lse are needed");
  if (!mask_fits(a)) return fail(PPN_E_INVALID, "ppn_loss_forward: a row of allowed has too few words");
  const ForwardPlan p = plan_forward(a);
  if (!a->workspace || a->workspace_bytes < p.bytes) return fail(PPN_E_INVALID, "ppn_loss_forward: the workspace is too small");
  if (!launches_fit(a, p)) return fail(PPN_E_INVALID, "loss: too many rows for as many actions and features");
  char* w = (char*)a->workspace;
  hipStream_t s = (hipStream_t)stream;
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    Operands o = {a->hidden, a->hidden_row, a->rows, a->weight, a->weight_row, a->actions, p.features_padded};
    if (p.hidden >= 0) {
      pad_rows<T>(a->hidden, a->hidden_row, a->rows, a->features, w + p.hidden, p.features_padded, s);
      o.A = w + p.hidden, o.lda = p.features_padded;
    }
    if (p.weight >= 0) {
      pad_rows<T>(a->weight, a->weight_row, a->actions, a->features, w + p.weight, p.features_padded, s);
      o.B = w + p.weight, o.ldb = p.features_padded;
    }
    const StatsArgs st = {a->allowed, a->allowed_row, (float2*)(w + p.partial), p.columns};
    const int64_t tm = ceil_div(a->rows, p.config.m), tn = ceil_div(a->actions, p.config.n);
    by_tile(p.config, [&](auto t) { loss_stats<T, decltype(t)::mi, decltype(t)::ni, decltype(t)::wm, decltype(t)::wn><<<dim3(tm * tn), dim3(256), 0, s>>>(o, st, tm, tn); });
    loss_join<T><<<dim3(ceil_div(a->rows, 16)), dim3(256), 0, s>>>(*a, st.partial, p.columns);
    return launched("ppn_loss_forward");
  });
}

extern "C" int64_t ppn_loss_backward_workspace(const ppn_loss_args* a) {
  if (int rc = check(a)) return rc;
  return plan_backward(a).bytes;
}

extern "C" int ppn_loss_backward(const ppn_loss_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  if (a->rows == 0) return fail(PPN_E_INVALID, "ppn_loss_backward: there are no rows");
  if (!a->hidden || !a->weight || !a->target || !a->loss || !a->lse || !a->dloss)
    return fail(PPN_E_INVALID, "ppn_loss_backward: hidden, weight, target, loss, lse and dloss are needed");
  if (!mask_fits(a)) return fail(PPN_E_INVALID, "ppn_loss_backward: a row of allowed has too few words");
  const BackwardPlan p = plan_backward(a);
  if (!a->workspace || a->workspace_bytes < p.bytes) return fail(PPN_E_INVALID, "ppn_loss_backward: the workspace is too small");
  if (!launches_fit(a, p)) return fail(PPN_E_INVALID, "loss: too many rows for as many actions and features");
  char* w = (char*)a->workspace;
  hipStream_t s = (hipStream_t)stream;
  float* scale = a->type == PPN_T_F16 ? (float*)(w + p.scale) : nullptr;
  return by_type(a->type, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    const void* hidden = a->hidden;
    const void* weight = a->weight;
    int64_t hidden_row = a->hidden_row, weight_row = a->weight_row;
    if (p.hidden >= 0) {
      pad_rows<T>(a->hidden, a->hidden_row, a->rows, a->features, w + p.hidden, p.features_padded, s);
      hidden = w + p.hidden, hidden_row = p.features_padded;
    }
    if (p.weight >= 0) {
      pad_rows<T>(a->weight, a->weight_row, a->actions, a->features, w + p.weight, p.features_padded, s);
      weight = w + p.weight, weight_row = p.features_padded;
    }
    const int64_t down = ceil_div(a->features, 64), hidden_across = ceil_div(p.rows_padded, 64), weight_across = ceil_div(p.actions_padded, 64);
    TransposeJob th = {a->hidden, a->hidden_row, a->rows, a->features, w + p.hidden_t, p.rows_padded, a->lse, (unsigned)hidden_across, a->dweight ? (unsigned)(hidden_across * down) : 0u};
    TransposeJob tw = {a->weight, a->weight_row, a->actions, a->features, w + p.weight_t, p.actions_padded, nullptr, (unsigned)weight_across, a->dhidden ? (unsigned)(weight_across * down) : 0u};
    if (scale) loss_scale<<<dim3(1), dim3(1024), 0, s>>>(a->dloss, a->lse, a->rows, scale);
    for (int64_t first = 0; first < a->actions; first += p.piece) {
      const int64_t n = a->actions - first < p.piece ? a->actions - first : p.piece, np = padded(n, 64);
      const Operands o = {hidden, hidden_row, a->rows, (const T*)weight + first * weight_row, weight_row, n, p.features_padded};
      const GradArgs g = {a->allowed, a->allowed_row, a->target, a->lse, a->loss, a->dloss, scale, w + p.dl, p.piece, w + p.dlt, p.rows_padded, first, p.rows_padded, np};
      const int64_t tm = ceil_div(a->rows, p.grad.m), tn = ceil_div(n, p.grad.n);
      by_large_tile(p.grad, [&](auto t) {
        loss_grad<T, decltype(t)::mi, decltype(t)::ni, decltype(t)::wm, decltype(t)::wn><<<dim3(tm * tn + th.blocks + tw.blocks), dim3(256), 0, s>>>(o, g, tm, tn, th, tw);
      });
      th.blocks = tw.blocks = 0;
      const int64_t across = ceil_div(a->features, p.sums.n);
      // (the last piece is shorter: a share that begins past its end adds nothing, and every slot has been written by the first piece)
      auto job = [&](const Operands& q, int64_t at, void* out, bool wanted, bool add) {
        const int64_t down = ceil_div(q.M, p.sums.m);
        return SumJob{q, (float*)(w + at), out, p.share, (unsigned)down, (unsigned)across, wanted ? (unsigned)(down * across * ceil_div(q.K, p.share)) : 0u, add};
      };
      const SumJob dh = job({w + p.dl, p.piece, a->rows, (const T*)(w + p.weight_t) + first, p.actions_padded, a->features, np}, p.dh,
                            p.direct_dh ? a->dhidden : nullptr, a->dhidden, first > 0);
      T* dw_out = (T*)a->dweight + (a->dweight ? first * a->features : 0);
      const SumJob dw = job({w + p.dlt, p.rows_padded, n, w + p.hidden_t, p.rows_padded, a->features, p.rows_padded}, p.dw,
                            p.direct_dw ? dw_out : nullptr, a->dweight, false);
      if (dh.blocks + dw.blocks)
        by_large_tile(p.sums, [&](auto t) { loss_sums<T, decltype(t)::mi, decltype(t)::ni, decltype(t)::wm, decltype(t)::wn><<<dim3(dh.blocks + dw.blocks), dim3(256), 0, s>>>(dh, dw, scale); });
      const bool last = first + p.piece >= a->actions;
      const FinishJob fh = {(const float*)(w + p.dh), p.dh_slots, last && a->dhidden && !p.direct_dh ? a->rows * a->features : 0, a->dhidden};
      const FinishJob fw = {(const float*)(w + p.dw), p.dw_slots, a->dweight && !p.direct_dw ? n * a->features : 0, dw_out};
      if (fh.count + fw.count) {
        const int64_t blocks = ceil_div(fh.count, 256);
        loss_finish<T><<<dim3(blocks + ceil_div(fw.count, 256)), dim3(256), 0, s>>>(fh, fw, blocks, scale);
      }
    }
    return launched("ppn_loss_backward");
  });
}
