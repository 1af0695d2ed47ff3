// Log-probabilities of given tokens straight from hidden states x [M, K] and the vocabulary projection w [N, K]: the logits
// z = x w^T / T are a matrix product whose tiles never leave the CU.
//   forward : where it saves rounds of tiles the rows that count are put together first; the product's epilogue reduces a tile to (max, sum of 2^D) per row and 48 or 64 columns (16 bytes of partial
//             results, there and back, for what would be 256 of bf16 logits), and picks the target's logit where its column passes; a second launch
//             joins a row's partial results.
//   backward: the product again (the logits were not kept), whose epilogue turns z into d(logits) = g ([j = t] - p_j) / T with the row's
//             maximum and sum from the forward; the gradients of x and w are two more products, where both are wanted large ones over the rows that count only.
//             d(logits) lies in memory until they are done, rounded to bf16 (2^-8 of each entry, as the gradient of bf16 logits is): the matrix instructions take bf16, and an fp32
//             entry would be two of them, each with products of its own.
// The logits are the products' fp32 sums here, never rounded to bf16.
#include <type_traits>
#include "log_probs.h"
#include "product_large.h"

namespace pico {
namespace {

// A wave has 16 J columns of a tile, which are a group: the width of a partial result.
constexpr int kFewJ = 4, kFewGroup = 16 * kFewJ, kLeastGroup = 48;
int groups_of(int64_t N, int width) { return static_cast<int>((N + width - 1) / width); }

// Partial results: (max, sum) of row r and group g at [r / 64][g][r % 64], so that a wave writes whole lines and a workgroup that joins reads neighbouring ones.
struct ScoreParams : LargeParams {
  const int64_t* targets;   // [M]
  f32x2* partial;
  float* target_logit;      // [M]
  int groups;
  float k;
  const int* count;       // rows that count, or NULL: all are taken as they lie
  const __bf16* packed;   // these rows put together, where some do not count
};
// the same value, of which the compiler does not know that it is (or it would keep what follows from it for all rows in registers)
__device__ __forceinline__ int hidden(int v) {
  asm volatile("" : "+v"(v));
  return v;
}
__device__ __forceinline__ float group_max(float v) {   // over the four lanes that have a row's columns
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return half_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
// (max, sum of 2^D) of 16 J columns of a row, 4 J of them in this lane: columns 16 j + 4 h + e, of which the first `cols` are there
template <int J>
__device__ __forceinline__ f32x2 score(f32x4 (&v)[J], int h, int cols, float k) {
  if (cols < 16 * J) {   // columns past the vocabulary
    const int left = hidden(cols - 4 * h);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = 16 * j + e < left ? v[j][e] : -INFINITY;
  }
  float m = v[0][0];
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) m = fmaxf(m, v[j][e]);
  m = group_max(m);
  // (the difference first: max k is off by up to its last bit, and so would all D be, which at a low temperature is more than a whole one)
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    float part = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) part += fast_exp2((v[j][e] - base) * k);
    s += part;
  }
  return {m, group_sum(s)};
}
// the target's logit to `to`, where its column is one of these (nearly always none of 16 rows' is); t: the target, two words
template <int J>
__device__ __forceinline__ void pick(const f32x4 (&v)[J], int2 t, int h, int col0, int vocab, bool live, float* to) {
  const int at = t.y == 0 && t.x >= 0 && t.x < vocab ? t.x - col0 : -1, place = at - 4 * h;
  if (__any(at >= 0 && at < 16 * J)) {
    float z = 0.f;
    bool here = false;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (place == 16 * j + e) { z = v[j][e]; here = true; }
      }
    if (here && live) *to = z;
  }
}

// 4 bytes per lane to LDS, as request16_to
template <int kPlus>
__device__ __forceinline__ void request4_to(uint32_t lds_off, u32x4 window, uint32_t off) {
  uint32_t aim;
  asm volatile("s_add_u32 %0, %1, %2\n\ts_nop 0\n\tbuffer_load_dword %3, %4, 0 offen lds"
               : "=&{m0}"(aim) : "s"(lds_off), "n"(kPlus), "v"(off), "s"(window) : "scc", "memory");
}

// Epilogue of the forward.  A lane holds columns 4 h ..+3 (h = lane / 16) of 16 consecutive ones, of row lane % 16 of 16: a row's
// columns meet over four lanes.  128 exponentials a lane at a quarter of the vector rate are most of it.
struct ScoreTile {
  using Params = ScoreParams;
  static constexpr bool kCounted = true;
  template <int TM>
  static __device__ __forceinline__ void count(Params& p) {
    if (p.count == nullptr) return;
    const int n = *p.count;
    if (n < p.M) p.a = p.packed;
    p.M = n;
    p.tiles_m = (n + TM - 1) / TM;
  }
  template <int I, int J> static constexpr int kStores = (I + 3) / 4;
  template <int I> static constexpr int kBegun = I / 2;   // 256 bytes each: 32 rows
  // the targets of the wave's rows, 8 bytes each, go to its rows region and are there long before the tile's end
  template <int I>
  static __device__ __forceinline__ void begin(const Params& p, const Unit& u, int wm, int lane, int wave, uint32_t lds_rows) {
    lane = hidden(lane);
    const int left = min(16 * I, p.M - u.m0 - wm);
    const u32x4 window = request_window(reinterpret_cast<uint64_t>(p.targets + u.m0 + wm), left > 0 ? left * 8u : 0u);
    wait_lds();
    each(std::make_integer_sequence<int, kBegun<I>>(), [&](auto piece) __attribute__((always_inline)) {
      request4_to<decltype(piece)::value * 256>(lds_rows, window, decltype(piece)::value * 256 + lane * 4);
    });
  }
  template <int I, int J>
  static __device__ __forceinline__ void tile(const Params& p, const Unit& u, int wm, int wn, int lane, const unsigned char* rows, f32x4 (&acc)[I][J]) {
    lane = hidden(lane);
    const int row0 = u.m0 + wm, col0 = u.n0 + wn, n = lane % 16, h = lane / 16, cols = p.N - col0;
    const float k = p.k;
    f32x2 mine = {0.f, 0.f};   // of row 64 q + lane
    const int live = p.M - row0;
    const u32x4 w = request_window(reinterpret_cast<uint64_t>(p.partial + (static_cast<int64_t>(row0 / 64) * p.groups + col0 / (16 * J)) * 64), 0x7ffffff0u);
    const buffer_rsrc window = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(w[0] | static_cast<uint64_t>(w[1]) << 32), 0, static_cast<int>(w[2]), static_cast<int>(w[3]));
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int row = 16 * i + n;
      pick(acc[i], *reinterpret_cast<const int2*>(rows + row * 8), h, col0, p.N, row < live, p.target_logit + row0 + row);
      const f32x2 ms = score(acc[i], h, cols, k);
      if (h == i % 4) mine = ms;
      if (i % 4 == 3 || i == I - 1) {
        const int r = i / 4 * 64 + lane, past = row0 % 64 + r;   // (the first row may lie inside a block of 64)
        const bool there = r < min(16 * I, live) && cols > 0;
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, mine), window, there ? (past / 64 * p.groups * 64 + past % 64) * 8 : static_cast<int>(0xfffffff0u), 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// Few rows (16 RB at most): what bounds them is reading w once.  A workgroup has 64 entries of the vocabulary, and its four waves a quarter of the contraction
// each, 128 bytes of a row at a time; operands come straight from memory in the layout of the products (x from the caches), a step's loads ahead of the step
// before's products, and the waves' sums meet in LDS.  Whole calls, us, in the product's tiles and here: 1 row of 2048 against 49152 52.5, 45.9 (4.4 TB/s), 16 rows 56.2,
// 48.4, 32 rows 52.3, 53.0; 24 x 576 18.5, 17.1; 32 x 4096 against 32000 79.0, 68.2.  Of 18 sizes the product's tiles took 0.87 to 1.84 of the time at 32 rows and
// 0.92 to 1.94 at 24; with 64 rows x would be read as often as w: they stay with the product.
template <int RB>
__global__ __launch_bounds__(256, 3) void score_few_kernel(const ScoreParams p) {
  __shared__ f32x4 sums[4][RB][kFewJ][kWave];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), n = lane % 16, h = lane / 16;
  const int col0 = blockIdx.x * kFewGroup, cols = p.N - col0;
  const char* w = reinterpret_cast<const char*>(p.b + static_cast<int64_t>(col0) * p.ldb);
  const char* x = reinterpret_cast<const char*>(p.a);
  uint32_t wo[kFewJ], xo[RB];   // (rows past the end read the last one)
#pragma unroll
  for (int j = 0; j < kFewJ; ++j) wo[j] = static_cast<uint32_t>(min(16 * j + n, cols - 1) * p.ldb * 2 + 16 * h);
#pragma unroll
  for (int b = 0; b < RB; ++b) xo[b] = static_cast<uint32_t>(min(16 * b + n, p.M - 1) * p.lda * 2 + 16 * h);
  struct Step {
    bf16x8 w[2][kFewJ], x[2][RB];
  };
  auto load = [&](Step& f, int step) __attribute__((always_inline)) {
    const char *wk = w + step * 128, *xk = x + step * 128;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int j = 0; j < kFewJ; ++j) f.w[s][j] = *reinterpret_cast<const bf16x8*>(wk + (wo[j] + 64u * s));
#pragma unroll
      for (int b = 0; b < RB; ++b) f.x[s][b] = *reinterpret_cast<const bf16x8*>(xk + (xo[b] + 64u * s));
    }
  };
  f32x4 acc[RB][kFewJ];
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int j = 0; j < kFewJ; ++j) acc[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Step& f) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int j = 0; j < kFewJ; ++j) acc[b][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.w[s][j], f.x[s][b], acc[b][j], 0, 0, 0);
  };
  const int whole = p.K / 64;
  Step one, two;
  int step = wave;
  if (step < whole) load(one, step);
  for (; step + 4 < whole; step += 8) {
    load(two, step + 4);
    __builtin_amdgcn_sched_barrier(0);
    multiply(one);
    if (step + 8 < whole) load(one, step + 8);
    __builtin_amdgcn_sched_barrier(0);
    multiply(two);
  }
  if (step < whole) multiply(one);
  if (p.K % 64 != 0 && wave == whole % 4) {   // the contraction's last piece, with zeros behind its end
    const char *wk = w + whole * 128, *xk = x + whole * 128;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bool in = whole * 64 + 32 * s + 8 * h < p.K;
#pragma unroll
      for (int j = 0; j < kFewJ; ++j) {
        one.w[s][j] = bf16x8{};
        if (in) one.w[s][j] = *reinterpret_cast<const bf16x8*>(wk + (wo[j] + 64u * s));
      }
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        one.x[s][b] = bf16x8{};
        if (in) one.x[s][b] = *reinterpret_cast<const bf16x8*>(xk + (xo[b] + 64u * s));
      }
    }
    multiply(one);
  }
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int j = 0; j < kFewJ; ++j) sums[wave][b][j][lane] = acc[b][j];
  __syncthreads();
  for (int b = wave; b < RB; b += 4) {
    f32x4 v[kFewJ];
#pragma unroll
    for (int j = 0; j < kFewJ; ++j) v[j] = (sums[0][b][j][lane] + sums[1][b][j][lane]) + (sums[2][b][j][lane] + sums[3][b][j][lane]);
    const int row = 16 * b + n;
    const bool live = row < p.M;
    const int2 t = live ? *reinterpret_cast<const int2*>(p.targets + row) : int2{-1, -1};
    pick(v, t, h, col0, p.N, live, p.target_logit + row);
    const f32x2 ms = score(v, h, cols, p.k);
    if (h == 0 && live) p.partial[static_cast<int64_t>(blockIdx.x) * 64 + row] = ms;
  }
}
constexpr int kFewRows = 32;

// ---- the rows that count, put together.  A prompt's and a padding's rows need no product; how many there are is known on the device only, so the product's
// workgroups look at the count and those past its tiles end.  position[row]: where a row went, -1 where it does not count.  Where all count x stays where it is.
// Every workgroup counts the rows in front of its own for itself (32 KB of targets for 4096 rows, from the caches): one launch, 3 - 4 us where all count.  Whole calls, us, all
// rows taken as they lie and put together, with all, 90 % and half of them counting: [4096 x 2048] against 49152 609, 611, 599, 324; [2000 x 4096] against 32000 391,
// 394, 394, 212; [3000 x 576] against 49152 155, 157, 154, 91.  In one or two rounds of tiles too few are saved: [1000 x 4096] against 32000 205, 208, 214, 161, [512 x 2048]
// against 49152 99, 102, 108, 103.
constexpr int kPackThreads = 1024, kLeastRows = 2 * kStep;
int pack_rows_of(int64_t M) { return static_cast<int>(std::max<int64_t>(16, (M + 255) / 256)); }   // a workgroup's (all workgroups' counting grows with M only)
__global__ __launch_bounds__(kPackThreads) void pack_rows_kernel(const __bf16* __restrict__ x, const int64_t* __restrict__ targets, int* __restrict__ position,
                                                                 int* __restrict__ count, int64_t* __restrict__ packed_targets, __bf16* __restrict__ packed, int M,
                                                                 int K, int vocab, int per, int64_t ignore_index) {
  constexpr int W = kPackThreads / kWave;
  __shared__ int all_of[W], before_of[W], to[kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, row0 = blockIdx.x * per;
  auto counts = [&](int64_t t) { return t != ignore_index && t >= 0 && t < vocab; };
  int all = 0, before = 0;
  constexpr int U = 4;   // targets requested together
  for (int first = threadIdx.x; first < M; first += U * kPackThreads) {
    int64_t t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) t[u] = first < M - u * kPackThreads ? targets[first + u * kPackThreads] : ignore_index;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = counts(t[u]);
      all += in;
      before += in && first + u * kPackThreads < row0;
    }
  }
#pragma unroll
  for (int off = kWave / 2; off > 0; off /= 2) {
    all += __shfl_xor(all, off, kWave);
    before += __shfl_xor(before, off, kWave);
  }
  if (lane == 0) { all_of[wave] = all; before_of[wave] = before; }
  __syncthreads();
  all = before = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) { all += all_of[i]; before += before_of[i]; }
  if (blockIdx.x == 0 && threadIdx.x == 0) *count = all;
  if (blockIdx.x == 0 && all < M)   // zeros up to the least contraction of the gradient of w
    for (int r = all + wave; r < min(kLeastRows, M); r += W)
      for (int piece = lane; piece < K / 8; piece += kWave) reinterpret_cast<u32x4*>(packed + static_cast<int64_t>(r) * K)[piece] = u32x4{0u, 0u, 0u, 0u};
  const int last = min(row0 + per, M);
  for (int first = row0; first < last; first += kWave) {   // 64 rows at a time
    if (wave == 0) {
      const int row = first + lane;
      const int64_t t = row < last ? targets[row] : ignore_index;
      const bool in = counts(t);
      const auto which = __ballot(in);
      const int at = in ? before + __popcll(which & ((1ull << lane) - 1)) : -1;
      before += __popcll(which);
      to[lane] = at;
      if (row < last) position[row] = at;
      if (in) packed_targets[at] = t;
    }
    __syncthreads();
    if (all != M)
      for (int r = wave; r < kWave; r += W) {
        if (to[r] < 0) continue;
        const u32x4* from = reinterpret_cast<const u32x4*>(x + static_cast<int64_t>(first + r) * K);
        u32x4* there = reinterpret_cast<u32x4*>(packed + static_cast<int64_t>(to[r]) * K);
        constexpr int P = 4;   // pieces requested together
        for (int piece = lane; piece < K / 8; piece += P * kWave) {
          u32x4 v[P];
#pragma unroll
          for (int i = 0; i < P; ++i)
            if (piece + i * kWave < K / 8) v[i] = from[piece + i * kWave];
#pragma unroll
          for (int i = 0; i < P; ++i)
            if (piece + i * kWave < K / 8) there[piece + i * kWave] = v[i];
        }
      }
    __syncthreads();
  }
}

// (log S as a whole, with the target's own 1 in it: a nearly certain token's log-probability is off by 2^-24, not by 2^-16 of itself.  The target is not left out of a group's sum, where
// its column would have to be told from 48 or 64 others.)
// A workgroup joins the partial results of kJoinRows rows: a row's groups are dealt to kSlices threads.  3.3 us at 24 rows of 49152 (one partial result after the
// other: 4.8), 7 at 4096; 8 rows of 128 slices take 0.4 us less at up to 32 rows, 3 more from 3000 on.
constexpr int kJoinRows = 16, kSlices = 64;
__global__ __launch_bounds__(kJoinRows * kSlices) void join_kernel(const f32x2* __restrict__ partial, const float* __restrict__ target_logit,
                                                                   const int64_t* __restrict__ targets, float* __restrict__ log_probs,
                                                                   f32x2* __restrict__ max_sum, const int* __restrict__ position, int M, int groups, int vocab, float k, float inv_t,
                                                                   int64_t ignore_index) {
  constexpr int kWaves = kSlices * kJoinRows / kWave, kOf = kWave / kJoinRows;   // a wave has kOf slices of kJoinRows rows
  __shared__ f32x2 share[kWaves][kJoinRows];
  const int r = threadIdx.x % kJoinRows, slice = threadIdx.x / kJoinRows, row = blockIdx.x * kJoinRows + r;
  const bool writes = slice == 0 && row < M;
  const int at = row >= M ? -1 : position != nullptr ? position[row] : row;   // (-1: it does not count and was left out)
  const int64_t t = writes ? targets[row] : 0;
  const float z = writes && at >= 0 ? target_logit[at] : 0.f;
  Gather<false> g;
  if (at >= 0) {
    constexpr int U = 6;   // partial results requested together
    const f32x2* of = partial + static_cast<int64_t>(at / 64) * groups * 64 + at % 64;
    for (int first = slice; first < groups; first += U * kSlices) {
      f32x2 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int group = first + u * kSlices;
        v[u] = group < groups ? of[group * 64] : f32x2{-INFINITY, 0.f};
      }
      g.meet(v, k);
    }
  }
  // a row's slices meet over lanes, waves (in LDS) and lanes
  auto over_lanes = [&] {
#pragma unroll
    for (int off = kJoinRows; off < kWave; off *= 2) {
      const f32x2 other[1] = {{__shfl_xor(g.zmax, off, kWave), __shfl_xor(g.s, off, kWave)}};
      g.meet(other, k);
    }
  };
  over_lanes();
  if (threadIdx.x % kWave < kJoinRows) share[threadIdx.x / kWave][r] = f32x2{g.zmax, g.s};
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  f32x2 waves[kWaves / kOf];
#pragma unroll
  for (int i = 0; i < kWaves / kOf; ++i) waves[i] = share[slice * (kWaves / kOf) + i][r];
  g = {};
  g.meet(waves, k);
  over_lanes();
  if (writes) {
    const bool counts = t != ignore_index && t >= 0 && t < vocab;
    log_probs[row] = counts ? (z - g.zmax) * inv_t - logf(g.s) : 0.f;
    if (max_sum != nullptr) max_sum[row] = at >= 0 ? f32x2{g.m, g.s} : f32x2{0.f, 1.f};
  }
}

// ---- backward
// a row as the epilogue needs it: p_j = 2^(k (z_j - max) - log2 S) (k max + log2 S as one number would be off by up to its last bit, and so would all p be); g = the
// gradient of its log-probability over T; the target's column, -1 where the row does not count (its gradient is 0, whatever its logits hold)
struct GradRow {
  float max, log2_s, g;
  int target;
};
__global__ void grad_rows_kernel(const f32x2* __restrict__ max_sum, const float* __restrict__ dlog_probs, const int64_t* __restrict__ targets,
                                 GradRow* __restrict__ out, const int* __restrict__ position, const int* __restrict__ count, int M, int vocab, float k, float inv_t,
                                 int64_t ignore_index) {
  const int row = blockIdx.x * blockDim.x + threadIdx.x;
  if (row >= M) return;
  const int at = position != nullptr ? position[row] : row;
  if (count != nullptr && row >= *count && row < kLeastRows) out[row] = {0.f, 0.f, 0.f, -1};   // (behind the rows that are put together)
  if (at < 0) return;
  const int64_t t = targets[row];
  const bool counts = t != ignore_index && t >= 0 && t < vocab && dlog_probs[row] != 0.f;
  const f32x2 ms = max_sum[row];
  const float g = ms[1] > 0.f ? dlog_probs[row] * inv_t : NAN;   // (a row whose logits are no numbers: p is held to 0 .. 1 below)
  out[at] = {ms[0], log2f(ms[1]), counts ? g : 0.f, counts ? static_cast<int>(t) : -1};
}

struct GradParams : LargeParams {
  const GradRow* grad_rows;   // [M]
  int ldc;
  float k;
  const int* count;           // (as in ScoreParams)
  const __bf16* packed;
};
struct GradTile {
  using Params = GradParams;
  static constexpr bool kCounted = true;
  template <int TM>
  static __device__ __forceinline__ void count(Params& p) {
    if (p.count == nullptr) return;
    const int n = *p.count;
    if (n < p.M) p.a = p.packed;
    p.M = max(n, kLeastRows);
    p.tiles_m = (p.M + TM - 1) / TM;
  }
  template <int I, int J> static constexpr int kStores = I * ((J + 3) / 4) * 2;
  template <int I> static constexpr int kBegun = (I + 3) / 4;   // 1 KiB each: 64 rows
  template <int I>
  static __device__ __forceinline__ void begin(const Params& p, const Unit& u, int wm, int lane, int wave, uint32_t lds_rows) {
    lane = hidden(lane);
    const int left = min(16 * I, p.M - u.m0 - wm);
    const u32x4 window = request_window(reinterpret_cast<uint64_t>(p.grad_rows + u.m0 + wm), left > 0 ? left * 16u : 0u);
    wait_lds();
    request16_to<0>(lds_rows, window, lane * 16);
    if constexpr (kBegun<I> > 1) request16_to<1024>(lds_rows, window, 1024 + lane * 16);
    static_assert(kBegun<I> <= 2);
  }
  template <int I, int J>
  static __device__ __forceinline__ void tile(const Params& p, const Unit& u, int wm, int wn, int lane, unsigned char* rows, f32x4 (&acc)[I][J]) {
    lane = hidden(lane);
    const int col0 = u.n0 + wn, n = lane % 16, h = lane / 16, cols = p.N - col0;
    const float k = p.k;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const GradRow r = *reinterpret_cast<const GradRow*>(rows + (16 * i + n) * 16);
      const int at = r.target - col0 - 4 * h;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // (p is 1 at most also where the forward, up to 32 rows, added a logit up in another order and the temperature makes much of the difference; a modifier of the exponential)
          const float p = __builtin_amdgcn_fmed3f(fast_exp2(fmaf(acc[i][j][e] - r.max, k, -r.log2_s)), 0.f, 1.f), d = fmaf(-r.g, p, at == 16 * j + e ? r.g : 0.f);
          acc[i][j][e] = r.target >= 0 ? d : 0.f;
        }
      if (cols < 16 * J) {   // zeros in the columns that pad a row
        const int left = hidden(cols - 4 * h);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = 16 * j + e < left ? acc[i][j][e] : 0.f;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    store_tile<__bf16, I, J>(static_cast<__bf16*>(p.c), 0, p.M, p.ldc, p.ldc, p.streaming, u, wm, wn, lane, rows, acc);
  }
};

// ---- the two products with d(logits) of the rows that count, put together.  Both operands' rows that do not count are missing: the gradient of w is a shorter
// contraction, that of x has fewer rows.  The latter's contraction (the vocabulary) is cut into parts such that its tiles fill the GPU, which depends on the
// number of rows and is found where that is known; the parts' sums go to the rows' places in a launch of their own.  Forward and backward, us, with all rows in the
// backward's products and with those that count, all, 90 %, 60 % and 30 % of them: [2000 x 4096] against 32000 1609, 1594, 1456, 1318 and 1607, 1552, 1106, 675; [2800 x
// 576] against 49152 714, 703, 664, 613 and 704, 655, 490, 341; [512 x 4096] against 32000 485, 482, 482, 470 and 500, 485, 421, 363; [2048 x 1024] against 49152 705,
// 700, 640, 596 and 725, 699, 521, 393.
struct CountedParams : LargeParams {
  const int* count;
  const __bf16* packed;
  int rows;   // all
};
constexpr int kMostParts = 32;
constexpr int64_t kMostPartial = 1 << 25;   // fp32 sums in parts: two rounds of tiles
// (The product and the launch that sums the parts each find it for themselves, and find the same: over all numbers of tiles and bounds on q that can occur, cost rounded after each
// operation, contracted and exact choose alike.)
__device__ __forceinline__ int parts_of(int tiles, int n, int hidden) {
  int best = 1;
  float least = static_cast<float>((tiles + 255) / 256);
  for (int q = 2; q <= kMostParts && static_cast<int64_t>(q) * n * hidden <= kMostPartial; ++q) {
    const float cost = static_cast<float>((tiles * q + 255) / 256) / static_cast<float>(q) + 0.02f * static_cast<float>(q - 1);   // (a part's sums written and read)
    if (cost < least) least = cost, best = q;
  }
  return best;
}
struct InputGradTile : StoreTile<true> {   // a: d(logits), b: w; fp32 [parts, rows that count, hidden]
  using Params = CountedParams;
  static constexpr bool kCounted = true;
  template <int TM>
  static __device__ __forceinline__ void count(Params& p) {
    p.M = *p.count;
    p.tiles_m = (p.M + TM - 1) / TM;
    p.parts = parts_of(p.tiles_m * p.tiles_n, p.M, p.N);
  }
};
struct WeightGradTile : StoreTile<false> {   // a: d(logits), b: x
  using Params = CountedParams;
  static constexpr bool kCounted = true;
  template <int TM>
  static __device__ __forceinline__ void count(Params& p) {
    const int n = *p.count;
    if (n < p.rows) p.b = p.packed;
    p.K = max(n, kLeastRows);
  }
};
constexpr int kUnpackThreads = 256;
__global__ __launch_bounds__(kUnpackThreads) void unpack_rows_kernel(const float* __restrict__ partial, const int* __restrict__ position, const int* __restrict__ count,
                                                                     __bf16* __restrict__ dx, int rows, int K, int tile_rows, int tiles_n,
                                                                     const __bf16* __restrict__ dlogits, const __bf16* __restrict__ w, int ldd, int64_t ldw, int from_entry,
                                                                     int vocab) {
  const int pieces = K / 8, n = *count, parts = parts_of((n + tile_rows - 1) / tile_rows * tiles_n, n, K);
  const int64_t all = static_cast<int64_t>(rows) * pieces, id = static_cast<int64_t>(blockIdx.x) * kUnpackThreads + threadIdx.x;
  if (id >= all) return;
  const int64_t row = id / pieces, at = position[row], piece = id - row * pieces;
  f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
  if (at >= 0)
    for (int q = 0; q < parts; ++q) {
      const f32x4* from = reinterpret_cast<const f32x4*>(partial + ((static_cast<int64_t>(q) * n + at) * pieces + piece) * 8);
      lo += from[0];
      hi += from[1];
    }
  if (at >= 0)   // the vocabulary's last entries, of which no whole piece of 16 bytes is left
    for (int entry = from_entry; entry < vocab; ++entry) {
      const float g = static_cast<float>(dlogits[at * ldd + entry]);
      const bf16x8 of = *reinterpret_cast<const bf16x8*>(w + entry * ldw + piece * 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = fmaf(g, static_cast<float>(of[e]), lo[e]);
        hi[e] = fmaf(g, static_cast<float>(of[4 + e]), hi[e]);
      }
    }
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = static_cast<__bf16>(lo[e]);
    v[4 + e] = static_cast<__bf16>(hi[e]);
  }
  reinterpret_cast<bf16x8*>(dx)[id] = v;
}

// ---- the gradient of w from few rows (32 at most): d(logits)^T x has a contraction of one product, and what bounds it is writing dw once.  A wave keeps x's
// 128 columns in registers as operands and walks 16 rows of dw at a time, whose d(logits) it requests one step ahead.  Tile j's column c is column
// 32 (j / 2) + 8 (c / 4) + 4 (j % 2) + c % 4 of the 128, so that two tiles give a lane 16 bytes and four lanes 64 of a row.  us, the GEMM library and here: 16 rows of
// 2048 against 49152 66, 34 (5.9 TB/s), 32 rows 44, 36, 4 of 2112 182, 42, 32 of 1024 against 120000 94, 44.  (Where the package's other products take it, up to
// 576 or 1024 columns, they are 2 .. 10 us faster; 64 rows, two products, took 0.85 to 1.04 of the library's time.)
constexpr int kFewGradRows = 32, kGradJ = 8, kGradColumns = 16 * kGradJ, kGradWalk = 16;   // kGradWalk steps of 16 rows of dw
__global__ __launch_bounds__(256) void weight_grad_few_kernel(const __bf16* __restrict__ d, const __bf16* __restrict__ x, __bf16* __restrict__ dw, int M, int N, int K,
                                                              int64_t ldd, int64_t ldx) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, n = lane % 16, h = lane / 16;
  const int col0 = (blockIdx.x * 4 + wave) * kGradColumns, row0 = blockIdx.y * 16 * kGradWalk;
  if (col0 >= K) return;
  bf16x8 fx[kGradJ];
#pragma unroll
  for (int j = 0; j < kGradJ; ++j) {
    const int col = col0 + 32 * (j / 2) + 8 * (n / 4) + 4 * (j % 2) + n % 4;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int r = 8 * h + e;
      const __bf16 v = x[min(r, M - 1) * ldx + min(col, K - 1)];   // (no load hangs on a condition: they are requested together, 58 -> 35 us)
      fx[j][e] = r < M ? v : static_cast<__bf16>(0.f);
    }
  }
  auto load = [&](bf16x8& f, int row) __attribute__((always_inline)) {   // d(logits) of rows row .. row + 15 of dw (past M: beside zeros of x)
    const __bf16* from = d + min(row + n, N - 1);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = from[min(8 * h + e, M - 1) * ldd];
  };
  bf16x8 now, next;
  load(now, row0);
  const int last = min(row0 + 16 * kGradWalk, N);
  for (int row = row0; row < last; row += 16, now = next) {
    if (row + 16 < last) load(next, row + 16);
#pragma unroll
    for (int j = 0; j < kGradJ; j += 2) {
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
      const f32x4 v[2] = {__builtin_amdgcn_mfma_f32_16x16x32_bf16(fx[j], now, zero, 0, 0, 0), __builtin_amdgcn_mfma_f32_16x16x32_bf16(fx[j + 1], now, zero, 0, 0, 0)};
      bf16x8 out;
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = static_cast<__bf16>(v[e / 4][e % 4]);
      const int col = col0 + 16 * j + 8 * h;
      if (row + n < last && col < K) *reinterpret_cast<bf16x8*>(dw + static_cast<int64_t>(row + n) * K + col) = out;
    }
  }
}

// ---- x with zeros in the rows that do not count, for a gradient of w that is taken over all rows: theirs of d(logits) are 0, but 0 times what a padded row
// may hold (NaN, infinities) is not.  One read, one write: whole calls, us, without and with it, [4 x 2112] against 49152 178, 181, [32 x 2048] against 32000
// 132, 134, [511 x 4096] against 32000 481, 485; by itself 5.1 at [2000 x 4096], 11 at [4096 x 4096].
constexpr int kCountedThreads = 256;
__global__ __launch_bounds__(kCountedThreads) void counted_rows_kernel(const __bf16* __restrict__ x, const int64_t* __restrict__ targets, __bf16* __restrict__ out, int64_t all,
                                                                       int pieces, int64_t ldx, int vocab, int64_t ignore_index) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kCountedThreads + threadIdx.x;
  if (id >= all) return;
  const int64_t row = id / pieces, piece = id - row * pieces, t = targets[row];
  u32x4 v = {0u, 0u, 0u, 0u};
  if (t != ignore_index && t >= 0 && t < vocab) v = *reinterpret_cast<const u32x4*>(x + row * ldx + piece * 8);
  reinterpret_cast<u32x4*>(out)[id] = v;
}

template <int I, int J, typename Epilogue, bool kSlowA = false, bool kSlowB = false>
int launch(typename Epilogue::Params p, const char* fn, hipStream_t s) {
  using S = Shape<kSlowA, kSlowB, I, J>;
  static LdsOnce reserved;
  if (!reserve_lds_once(reserved, reinterpret_cast<const void*>(&product_large_kernel<kSlowA, kSlowB, I, J, Epilogue>), S::kLds))
    return fail(PICO_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS", fn, S::kLds);
  p.tiles_m = (p.M + S::TM - 1) / S::TM;
  p.tiles_n = (p.N + S::TN - 1) / S::TN;
  p.parts = 1;
  const int64_t units = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  p.streaming = units > 256;   // (as pico_product_large)
  // (the input gradient's parts are not known here)
  const unsigned grid = std::is_same_v<Epilogue, InputGradTile> ? 256u : static_cast<unsigned>(std::min<int64_t>(units, 256));
  hipLaunchKernelGGL((product_large_kernel<kSlowA, kSlowB, I, J, Epilogue>), dim3(grid), dim3(S::kThreads), S::kLds, s, p);
  return check_launch(fn);
}
// fn(rows / 32, columns / 64) of the tile whose rounds of 256 workgroups take the least time.  A round's time relative to 256 x 256, at [3000 x 2048] @
// [49152 x 2048]^T: 51.8 us, 192 x 256 41.5, 256 x 192 42.5, 128 x 256 32.9, 128 x 192 28.1 (256 x 128 was never the best).  Over 60 shapes of 40 .. 3000 rows,
// hidden sizes 232 .. 4008 and vocabularies 2392 .. 120696 the rule is within 2 % of the best tile; with one of 256 columns throughout it lost up to 19 %: us at
// [rows x 2048] @ [49152 x 2048]^T, 256 x 256 | 192 x 256 | 128 x 256 | 256 x 192 | 128 x 192:
//    128 rows  61.8 |  59.7 |  58.9 |  59.7 |  54.9
//    256 rows  69.0 |  91.6 |  89.7 |  64.9 |  80.6
//    300 rows 100.9 |  93.6 | 116.4 |  96.2 | 108.5
//    512 rows 109.9 | 129.6 | 120.4 | 100.8 | 139.5
//   1000 rows 165.9 | 206.7 | 221.0 | 180.6 | 261.1
template <typename Fn>
int with_tile(int64_t M, int64_t N, const Fn& fn) {
  static constexpr struct { int i, j; double round; } kTiles[] = {{8, 4, 1.}, {6, 4, 0.84}, {8, 3, 0.84}, {4, 4, 0.64}, {4, 3, 0.56}};
  int best = 0;
  double least = INFINITY;
  for (int t = 0; t < 5; ++t) {
    const int64_t tm = 32 * kTiles[t].i, tn = 64 * kTiles[t].j;
    const double cost = kTiles[t].round * static_cast<double>(((M + tm - 1) / tm * ((N + tn - 1) / tn) + 255) / 256);
    if (cost < least) least = cost, best = t;
  }
  using std::integral_constant;
  switch (best) {
    case 0: return fn(integral_constant<int, 8>(), integral_constant<int, 4>());
    case 1: return fn(integral_constant<int, 6>(), integral_constant<int, 4>());
    case 2: return fn(integral_constant<int, 8>(), integral_constant<int, 3>());
    case 3: return fn(integral_constant<int, 4>(), integral_constant<int, 4>());
    default: return fn(integral_constant<int, 4>(), integral_constant<int, 3>());
  }
}

template <typename T>
void take(char*& next, T*& part, int64_t n) {   // n of them, from a 16-byte boundary
  part = reinterpret_cast<T*>(next);
  next += (n * static_cast<int64_t>(sizeof(T)) + 15) / 16 * 16;
}
// what the forward keeps beside its results
struct Workspace {
  __bf16* packed;        // [rows, hidden]
  f32x2* partial;        // [rows / 64][groups][64]
  int64_t* targets;      // [rows], of the packed ones
  float* target_logit;   // [rows]
  int *position, *count; // [rows], [1]
  int64_t bytes;
  Workspace(void* at, int64_t rows, int64_t hidden, int64_t vocab) {
    char* next = static_cast<char*>(at);
    take(next, packed, rows > kFewRows ? rows * hidden : 0);
    take(next, partial, (rows + 63) / 64 * 64 * groups_of(vocab, kLeastGroup));
    take(next, targets, rows);
    take(next, target_logit, rows);
    take(next, position, rows);
    take(next, count, 1);
    bytes = next - static_cast<char*>(at);
  }
};

struct BackwardWorkspace {
  __bf16 *dlogits, *packed;   // [rows, vocab], [rows, hidden]: of those that count
  float* partial;             // [parts][rows that count][hidden]
  GradRow* grad_rows;         // [rows]
  int64_t* targets;           // [rows]
  int *position, *count;      // [rows], [1]
  int64_t bytes;
  BackwardWorkspace(void* at, int64_t rows, int64_t hidden, int64_t vocab) {
    char* next = static_cast<char*>(at);
    take(next, dlogits, rows * ((vocab + 7) / 8 * 8));
    take(next, packed, rows * hidden);
    take(next, partial, std::max(rows * hidden, kMostPartial));
    take(next, grad_rows, rows);
    take(next, targets, rows);
    take(next, position, rows);
    take(next, count, 1);
    bytes = next - static_cast<char*>(at);
  }
};

int check_linear(const char* fn, const void* x, const void* w, const int64_t* targets, int64_t M, int64_t K, int64_t N, int64_t ldx, int64_t ldw, float temperature) {
  if (M < 0 || N <= 0 || K % 8 != 0 || (M > 0 && !pico_product_large_takes(M, (N + 7) / 8 * 8, K, ldx, ldw, 0, 0, 1)))
    return fail(PICO_ERR_SHAPE, "%s: rows=%lld hidden=%lld vocab=%lld row pitches %lld, %lld (hidden a multiple of 8 over 64, pitches multiples of 8, a tile's rows span less than 2 GiB)",
                fn, static_cast<long long>(M), static_cast<long long>(K), static_cast<long long>(N), static_cast<long long>(ldx), static_cast<long long>(ldw));
  if (!(temperature > 0.f) || !(temperature <= 1e30f) || !(1.f / temperature <= 1e30f)) return fail(PICO_ERR_SHAPE, "%s: temperature %g must be positive and finite", fn, temperature);
  if (M == 0) return PICO_OK;
  if (!x || !w || !targets) return fail(PICO_ERR_NULL, "%s: x, w and targets are required", fn);
  if (!aligned16(x) || !aligned16(w) || reinterpret_cast<uintptr_t>(targets) % 8) return fail(PICO_ERR_ALIGN, "%s: x and w must be aligned to 16 bytes, targets to 8", fn);
  return PICO_OK;
}
void fill(LargeParams& p, const void* x, const void* w, int64_t M, int64_t K, int64_t N, int64_t ldx, int64_t ldw) {
  p.a = static_cast<const __bf16*>(x);
  p.b = static_cast<const __bf16*>(w);
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.lda = ldx;
  p.ldb = ldw;
}

}  // namespace
}  // namespace pico

using namespace pico;

extern "C" int64_t pico_linear_log_probs_workspace_bytes(int64_t rows, int64_t hidden, int64_t vocab) {
  if (rows < 0 || hidden < 0 || vocab < 0 || rows > 0x7fffffff || hidden > 0x7fffffff || vocab > 0x7fffffff) return -1;
  return Workspace(nullptr, rows, hidden, vocab).bytes;
}

extern "C" int pico_linear_log_probs_fwd(const void* x, const void* w, const int64_t* targets, float* log_probs, float* max_sum, int64_t rows, int64_t hidden,
                                         int64_t vocab, int64_t ldx, int64_t ldw, float temperature, int64_t ignore_index, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
  const char* fn = "pico_linear_log_probs_fwd";
  if (int rc = check_linear(fn, x, w, targets, rows, hidden, vocab, ldx, ldw, temperature)) return rc;
  if (rows == 0) return PICO_OK;
  if (!log_probs || !workspace) return fail(PICO_ERR_NULL, "%s: log_probs and workspace are required", fn);
  if (!aligned16(workspace) || reinterpret_cast<uintptr_t>(max_sum) % 8) return fail(PICO_ERR_ALIGN, "%s: workspace must be aligned to 16 bytes, max_sum to 8", fn);
  const Workspace of(workspace, rows, hidden, vocab);
  if (workspace_bytes < of.bytes)
    return fail(PICO_ERR_WORKSPACE, "%s: workspace of %lld bytes, needs %lld", fn, static_cast<long long>(workspace_bytes), static_cast<long long>(of.bytes));
  hipStream_t s = static_cast<hipStream_t>(stream);
  ScoreParams p = {};
  fill(p, x, w, rows, hidden, vocab, ldx, ldw);
  p.targets = targets;
  p.partial = of.partial;
  p.target_logit = of.target_logit;
  p.k = static_cast<float>(1.4426950408889634 / temperature);
  if (rows <= kFewRows) {
    p.groups = groups_of(vocab, kFewGroup);
    const dim3 grid(static_cast<unsigned>(p.groups)), threads(256);
    if (rows <= 16) hipLaunchKernelGGL(score_few_kernel<1>, grid, threads, 0, s, p);
    else hipLaunchKernelGGL(score_few_kernel<2>, grid, threads, 0, s, p);
  } else {
    const int rc = with_tile(rows, vocab, [&](auto i, auto j) {
      constexpr int I = decltype(i)::value, J = decltype(j)::value;
      p.groups = groups_of(vocab, 16 * J);
      // (rows with gaps between them are left to the product.  hidden x vocab: a row's product takes 40 times as long as its part of the packing, or longer)
      if (vocab * hidden >= (1 << 23) && (rows + 32 * I - 1) / (32 * I) * ((vocab + 64 * J - 1) / (64 * J)) > 2 * 256 && ldx == hidden) {
        const int per = pack_rows_of(rows);
        hipLaunchKernelGGL(pack_rows_kernel, dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(kPackThreads), 0, s, p.a, targets, of.position, of.count,
                           of.targets, of.packed, p.M, p.K, p.N, per, ignore_index);
        p.count = of.count;
        p.packed = of.packed;
        p.targets = of.targets;
      }
      return launch<I, J, ScoreTile>(p, fn, s);
    });
    if (rc) return rc;
  }
  hipLaunchKernelGGL(join_kernel, dim3(static_cast<unsigned>((rows + kJoinRows - 1) / kJoinRows)), dim3(kJoinRows * kSlices), 0, s, p.partial, p.target_logit, targets,
                     log_probs, reinterpret_cast<f32x2*>(max_sum), p.count ? of.position : nullptr, p.M, p.groups, p.N, p.k, 1.f / temperature, ignore_index);
  return check_launch(fn);
}

extern "C" int pico_linear_log_probs_dlogits(const void* x, const void* w, const int64_t* targets, const float* max_sum, const float* dlog_probs, void* dlogits,
                                             int64_t rows, int64_t hidden, int64_t vocab, int64_t ldx, int64_t ldw, int64_t ldd, float temperature,
                                             int64_t ignore_index, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "pico_linear_log_probs_dlogits";
  if (int rc = check_linear(fn, x, w, targets, rows, hidden, vocab, ldx, ldw, temperature)) return rc;
  if (ldd < vocab || ldd % 8 != 0 || ldd >= vocab + 8) return fail(PICO_ERR_STRIDE, "%s: row pitch %lld of dlogits must be vocab, rounded up to a multiple of 8", fn, static_cast<long long>(ldd));
  if (rows == 0) return PICO_OK;
  if (!max_sum || !dlog_probs || !dlogits || !workspace) return fail(PICO_ERR_NULL, "%s: max_sum, dlog_probs, dlogits and workspace are required", fn);
  if (!aligned16(dlogits) || !aligned16(workspace) || reinterpret_cast<uintptr_t>(max_sum) % 8)
    return fail(PICO_ERR_ALIGN, "%s: dlogits and workspace must be aligned to 16 bytes, max_sum to 8", fn);
  if (workspace_bytes < rows * 16) return fail(PICO_ERR_WORKSPACE, "%s: workspace of %lld bytes, needs 16 per row", fn, static_cast<long long>(workspace_bytes));
  hipStream_t s = static_cast<hipStream_t>(stream);
  GradParams p = {};
  fill(p, x, w, rows, hidden, vocab, ldx, ldw);
  p.k = static_cast<float>(1.4426950408889634 / temperature);
  GradRow* of = static_cast<GradRow*>(workspace);
  hipLaunchKernelGGL(grad_rows_kernel, dim3(static_cast<unsigned>((rows + 255) / 256)), dim3(256), 0, s, reinterpret_cast<const f32x2*>(max_sum), dlog_probs, targets, of,
                     nullptr, nullptr, p.M, p.N, p.k, 1.f / temperature, ignore_index);
  p.c = dlogits;
  p.ldc = static_cast<int>(ldd);
  p.grad_rows = of;
  return with_tile(rows, vocab, [&](auto i, auto j) { return launch<decltype(i)::value, decltype(j)::value, GradTile>(p, fn, s); });
}

// The whole backward, of the rows that count, where it is worth it: two rows of tiles, tiles of the gradient of w that fill the GPU twice, and of that of x enough that
// 32 parts of them fill it when few rows count (9 tiles, [600 x 576], took 391 us instead of 200 with a quarter of the parts).
extern "C" int64_t pico_linear_log_probs_bwd_workspace_bytes(int64_t rows, int64_t hidden, int64_t vocab) {
  const int64_t tiles_n = (hidden + 255) / 256, pitch = (vocab + 7) / 8 * 8, whole = vocab / 8 * 8;
  if (rows < 512 || hidden <= 0 || whole < 64 * 2 * kMostParts || vocab * hidden < (1 << 23) || (vocab + 255) / 256 * tiles_n < 512 ||
      (rows + 255) / 256 * tiles_n < 32 ||
      !pico_product_large_takes(rows, pitch, hidden, hidden, hidden, 0, 0, 1) || !pico_product_large_takes(rows, hidden, whole, pitch, hidden, 0, 1, kMostParts) ||
      !pico_product_large_takes(pitch, hidden, rows, pitch, hidden, 1, 1, 1) || rows * hidden > (int64_t{1} << 31))
    return 0;
  return BackwardWorkspace(nullptr, rows, hidden, vocab).bytes;
}

extern "C" int pico_linear_log_probs_bwd(const void* x, const void* w, const int64_t* targets, const float* max_sum, const float* dlog_probs, void* dx, void* dw,
                                         int64_t rows, int64_t hidden, int64_t vocab, int64_t ldw, float temperature, int64_t ignore_index, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
  const char* fn = "pico_linear_log_probs_bwd";
  if (int rc = check_linear(fn, x, w, targets, rows, hidden, vocab, hidden, ldw, temperature)) return rc;
  const int64_t bytes = pico_linear_log_probs_bwd_workspace_bytes(rows, hidden, vocab);
  const int64_t pitch = (vocab + 7) / 8 * 8, whole = vocab / 8 * 8;   // d(logits)' rows end in zeros up to pitch; whole pieces of 16 bytes
  if (bytes <= 0 || !pico_product_large_takes(rows, hidden, whole, pitch, ldw, 0, 1, kMostParts))
    return fail(PICO_ERR_SHAPE, "%s: rows=%lld hidden=%lld vocab=%lld (pitch of w %lld): pico_linear_log_probs_dlogits and two products take these", fn,
                static_cast<long long>(rows), static_cast<long long>(hidden), static_cast<long long>(vocab), static_cast<long long>(ldw));
  if (!max_sum || !dlog_probs || !dx || !dw || !workspace) return fail(PICO_ERR_NULL, "%s: max_sum, dlog_probs, dx, dw and workspace are required", fn);
  if (!aligned16(dx) || !aligned16(dw) || !aligned16(workspace) || reinterpret_cast<uintptr_t>(max_sum) % 8)
    return fail(PICO_ERR_ALIGN, "%s: dx, dw and workspace must be aligned to 16 bytes, max_sum to 8", fn);
  if (workspace_bytes < bytes) return fail(PICO_ERR_WORKSPACE, "%s: workspace of %lld bytes, needs %lld", fn, static_cast<long long>(workspace_bytes), static_cast<long long>(bytes));
  const BackwardWorkspace of(workspace, rows, hidden, vocab);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const float inv_t = 1.f / temperature;
  GradParams g = {};
  fill(g, x, w, rows, hidden, vocab, hidden, ldw);
  g.k = static_cast<float>(1.4426950408889634 / temperature);
  const int per = pack_rows_of(rows);
  hipLaunchKernelGGL(pack_rows_kernel, dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(kPackThreads), 0, s, g.a, targets, of.position, of.count, of.targets,
                     of.packed, g.M, g.K, g.N, per, ignore_index);
  hipLaunchKernelGGL(grad_rows_kernel, dim3(static_cast<unsigned>((rows + 255) / 256)), dim3(256), 0, s, reinterpret_cast<const f32x2*>(max_sum), dlog_probs, targets,
                     of.grad_rows, of.position, of.count, g.M, g.N, g.k, inv_t, ignore_index);
  g.c = of.dlogits;
  g.ldc = static_cast<int>(pitch);
  g.grad_rows = of.grad_rows;
  g.count = of.count;
  g.packed = of.packed;
  if (int rc = with_tile(rows, vocab, [&](auto i, auto j) { return launch<decltype(i)::value, decltype(j)::value, GradTile>(g, fn, s); })) return rc;
  // gradient of x: [rows that count, vocab] @ [vocab, hidden]; of w: [vocab, rows that count] @ [rows that count, hidden]
  CountedParams p = {};
  fill(p, of.dlogits, w, rows, whole, hidden, pitch, ldw);
  p.c = of.partial;
  p.count = of.count;
  p.rows = static_cast<int>(rows);
  CountedParams q = {};
  fill(q, of.dlogits, x, pitch, rows, hidden, pitch, hidden);
  q.c = dw;
  q.count = of.count;
  q.packed = of.packed;
  q.rows = p.rows;
  // (columns of 192 where they leave less over: hidden 576)
  const bool narrow = (hidden + 191) / 192 * 84 < (hidden + 255) / 256 * 100;
  if (int rc = narrow ? launch<8, 3, InputGradTile, false, true>(p, fn, s) : launch<8, 4, InputGradTile, false, true>(p, fn, s)) return rc;
  const int tn = narrow ? 192 : 256;
  hipLaunchKernelGGL(unpack_rows_kernel, dim3(static_cast<unsigned>((rows * (hidden / 8) + kUnpackThreads - 1) / kUnpackThreads)), dim3(kUnpackThreads), 0, s, of.partial,
                     of.position, of.count, static_cast<__bf16*>(dx), p.rows, static_cast<int>(hidden), 256, static_cast<int>((hidden + tn - 1) / tn), of.dlogits, p.b, g.ldc, ldw,
                     static_cast<int>(whole), static_cast<int>(vocab));
  return narrow ? launch<8, 3, WeightGradTile, true, true>(q, fn, s) : launch<8, 4, WeightGradTile, true, true>(q, fn, s);
}

extern "C" int pico_weight_grad_few(const void* d, const void* x, void* dw, int64_t rows, int64_t out, int64_t in, int64_t ldd, int64_t ldx, void* stream) {
  const char* fn = "pico_weight_grad_few";
  if (rows < 1 || rows > kFewGradRows || out < 1 || out > 0x7fffffff / 256 || in < 8 || in % 8 != 0 || in > 0x7fffffff / 256)
    return fail(PICO_ERR_SHAPE, "%s: rows=%lld (1 .. %d) out=%lld in=%lld (a multiple of 8)", fn, static_cast<long long>(rows), kFewGradRows, static_cast<long long>(out),
                static_cast<long long>(in));
  if (ldd < out || ldx < in) return fail(PICO_ERR_STRIDE, "%s: row pitches %lld, %lld are less than the rows", fn, static_cast<long long>(ldd), static_cast<long long>(ldx));
  if (!d || !x || !dw) return fail(PICO_ERR_NULL, "%s: d, x and dw are required", fn);
  if (reinterpret_cast<uintptr_t>(d) % 2 || reinterpret_cast<uintptr_t>(x) % 2 || !aligned16(dw)) return fail(PICO_ERR_ALIGN, "%s: dw must be aligned to 16 bytes, d and x to their elements", fn);
  const dim3 grid(static_cast<unsigned>((in + 4 * kGradColumns - 1) / (4 * kGradColumns)), static_cast<unsigned>((out + 16 * kGradWalk - 1) / (16 * kGradWalk)));
  hipLaunchKernelGGL(weight_grad_few_kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const __bf16*>(d), static_cast<const __bf16*>(x),
                     static_cast<__bf16*>(dw), static_cast<int>(rows), static_cast<int>(out), static_cast<int>(in), ldd, ldx);
  return check_launch(fn);
}

extern "C" int pico_linear_log_probs_counted(const void* x, const int64_t* targets, void* out, int64_t rows, int64_t hidden, int64_t vocab, int64_t ldx,
                                             int64_t ignore_index, void* stream) {
  const char* fn = "pico_linear_log_probs_counted";
  constexpr int64_t kMost = 0x7fffffff;
  // (a launch has fewer than 2^32 threads)
  if (rows < 0 || rows > kMost || hidden < 8 || hidden > kMost || hidden % 8 != 0 || vocab < 1 || vocab > kMost || rows * (hidden / 8) > 0xffffffffll - kCountedThreads)
    return fail(PICO_ERR_SHAPE, "%s: rows=%lld hidden=%lld (a multiple of 8) vocab=%lld", fn, static_cast<long long>(rows), static_cast<long long>(hidden), static_cast<long long>(vocab));
  if (ldx < hidden || ldx % 8 != 0) return fail(PICO_ERR_STRIDE, "%s: row pitch %lld must be a multiple of 8 and no less than a row", fn, static_cast<long long>(ldx));
  if (rows == 0) return PICO_OK;
  if (!x || !targets || !out) return fail(PICO_ERR_NULL, "%s: x, targets and out are required", fn);
  if (!aligned16(x) || !aligned16(out) || reinterpret_cast<uintptr_t>(targets) % 8) return fail(PICO_ERR_ALIGN, "%s: x and out must be aligned to 16 bytes, targets to 8", fn);
  const int64_t all = rows * (hidden / 8);
  hipLaunchKernelGGL(counted_rows_kernel, dim3(static_cast<unsigned>((all + kCountedThreads - 1) / kCountedThreads)), dim3(kCountedThreads), 0, static_cast<hipStream_t>(stream),
                     static_cast<const __bf16*>(x), targets, static_cast<__bf16*>(out), all, static_cast<int>(hidden / 8), ldx, static_cast<int>(vocab), ignore_index);
  return check_launch(fn);
}
