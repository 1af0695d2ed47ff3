// What the operators on log-probabilities of given tokens share: rows of logits that may start at any element, the statistics
// of a row, and the gradient that follows from them.
//   D_j = (logits_j - max) k, k = log2(e) / T: the logits' distances from the largest over T, in the log2 domain
//   S = sum 2^D_j,  p_j = 2^D_j / S,  log p_t = (logits_t - max) / T - ln S,  H = ln S - ln2 / S sum 2^D_j D_j
// (The difference first: logits k - max k is an instruction less, but overflows for the lowest value of a type, which masks are made
// of, and rounds every D by the last bit of max k.)
#pragma once
#include "common.h"

namespace pico {
namespace {

// (-1000 in the log2 domain is 0 for exp2, and 0 x -1000 is 0 where 0 x -inf would not be a number)
constexpr float kFloor = -1000.f;

struct LogitsArgs {
  const void* data;
  int64_t batch_stride, row_stride;   // elements
  int seq, vocab;
  float k, inv_t;                     // log2(e) / T, 1 / T
};
template <typename V> struct Strided {   // a value per row: [batch, seq] with any strides, 0 among them
  const V* data;
  int64_t batch_stride, row_stride;
  __device__ __forceinline__ V at(int64_t b, int64_t s) const { return data[b * batch_stride + s * row_stride]; }
};
using TokenArgs = Strided<int64_t>;
using ValueArgs = Strided<float>;

// A row: `head` elements up to the first 16-byte boundary, nvec pieces of 16 bytes, `tail` elements.  Head and tail together are
// fewer than two pieces: thread i < 8 has element i of the head, thread 8 + i element i of the tail.
template <typename T>
struct Row {
  static constexpr int V = io<T>::kVec;
  const T* x;      // the row
  const T* body;   // its first whole piece
  int head, nvec, edge;   // edge: this thread's element of head or tail, -1: none
  int inside;             // pieces between the line of 128 bytes that `body` lies in and body
  __device__ __forceinline__ Row(const void* data, int64_t offset, int vocab) {
    x = static_cast<const T*>(data) + offset;
    const int past = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    head = min(past ? V - past : 0, vocab);
    nvec = (vocab - head) / V;
    body = x + head;
    inside = static_cast<int>(reinterpret_cast<uintptr_t>(body) % 128 / 16);
    const int tail = vocab - head - nvec * V, i = threadIdx.x;
    edge = i < head ? i : i >= 8 && i - 8 < tail ? vocab - tail + i - 8 : -1;
  }
  // The thread's first piece; the others follow NT apart.  A wave's accesses are whole lines: stores of parts of lines past the caches are slow ([3, 777,
  // 32001] fp32 backward 119 -> 107 us).  (The first lanes of a row that starts inside a line come a round later.)
  template <int NT>
  __device__ __forceinline__ int first() const {
    const int v = static_cast<int>(threadIdx.x) - inside;
    return v < 0 ? v + NT : v;
  }
};

// What a row's statistics are gathered in, one element or piece after the other.
template <bool kEntropy>
struct Gather {
  float zmax = -INFINITY, m = 0.f, s = 0.f, w = 0.f;   // m: zmax, or 0 where nothing but -inf was there
  // to another maximum, no smaller than this one (no product here is taken into a sum unrounded: where lanes exchange sums, each would have another)
  __device__ __forceinline__ void rise(float to, float k) {
#pragma clang fp contract(off)
    const float shift = zmax == -INFINITY ? 0.f : fmaxf((zmax - to) * k, kFloor), c = fast_exp2(shift);
    if constexpr (kEntropy) w = c * (w + shift * s);
    s *= c;
    zmax = to;
    m = to == -INFINITY ? 0.f : to;
  }
  template <int N>
  __device__ __forceinline__ void meet(const f32x2 (&others)[N], float k) {   // (max, sum) gathered elsewhere (no entropy)
    float top = zmax;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, others[i][0]);
    rise(top, k);
#pragma unroll
    for (int i = 0; i < N; ++i) s += others[i][1] * fast_exp2(others[i][0] == -INFINITY ? 0.f : fmaxf((others[i][0] - top) * k, kFloor));
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&e)[N], float k) {
    float top = e[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, e[i]);
    if (top > zmax) rise(top, k);
    take(e, k);
  }
  // none over the maximum.  A piece's sum first: beside a certain token's 1 the others are added one by one with an error of 2^-24 each, and ln S is what they sum to.
  template <int N>
  __device__ __forceinline__ void take(const float (&e)[N], float k) {
    float ps = 0.f, pw = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = (e[i] - m) * k, p = fast_exp2(d);
      ps += p;
      if constexpr (kEntropy) pw = fmaf(p, fmaxf(d, kFloor), pw);
    }
    s += ps;
    if constexpr (kEntropy) w += pw;
  }
};

// The target's logit joins what was gathered of the others, and its log-probability.  Where it is the largest that is -ln(1 + the others), which keeps its relative
// accuracy however certain the token is; a sum that held the 1 from the beginning would have lost it.  (p - 1 there is 0, or not a number where the target is +inf.)
template <bool kEntropy>
__device__ __forceinline__ float with_target(Gather<kEntropy>& g, float xt, float k, float inv_t) {
  g.rise(fmaxf(g.zmax, xt), k);
  const float d = (xt - g.m) * k, p = fast_exp2(d), others = g.s;
  g.s = others + p;
  if constexpr (kEntropy) g.w = fmaf(p, fmaxf(d, kFloor), g.w);
  return xt == g.m ? -log1pf(others + (p - 1.f)) : (xt - g.m) * inv_t - logf(g.s);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, kWave));
  return v;
}

// A workgroup's gathered shares as one, for every thread.  `share`: 3 floats a wave of LDS.  A lane reads one wave's share and the lanes exchange them: read
// whole by every lane they would take three registers a wave, beside a row that is held in registers too many.
template <int NT, bool kEntropy>
__device__ __forceinline__ void join(Gather<kEntropy>& g, float k, float (*share)[3]) {
  constexpr int W = NT / kWave;
  g.rise(wave_max(g.zmax), k);
  g.s = wave_sum(g.s);
  if constexpr (kEntropy) g.w = wave_sum(g.w);
  if constexpr (W > 1) {
    const int wave = threadIdx.x / kWave, of = threadIdx.x % W;
    if (threadIdx.x % kWave == 0) { share[wave][0] = g.zmax; share[wave][1] = g.s; share[wave][2] = g.w; }
    __syncthreads();
    g.zmax = share[of][0];
    g.s = share[of][1];
    if constexpr (kEntropy) g.w = share[of][2];
    float top = g.zmax;
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
    g.rise(top, k);
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) {
      g.s += __shfl_xor(g.s, off, kWave);
      if constexpr (kEntropy) g.w += __shfl_xor(g.w, off, kWave);
    }
  }
}

// The gradient of a (log p_t) + b H in one row: g_j = 2^D_j (alpha + beta D_j) + [j = t] hot, with the 1 / T of z.
//   d log p_t / dz_j = [j = t] - p_j,  dH / dz_j = -p_j (ln p_j + H),  ln p_j = ln2 D_j - ln S
struct Slope {
  float alpha, beta, hot;
};
template <bool kEntropy>
__device__ __forceinline__ Slope slope(float a, float b, float s, float H, float inv_t) {
  const float scale = inv_t / s;
  Slope r = {-a * scale, 0.f, a * inv_t};
  if constexpr (kEntropy) {
    r.alpha -= b * (H - logf(s)) * scale;
    r.beta = -b * kLn2 * scale;
  }
  return r;
}
template <bool kEntropy>
__device__ __forceinline__ float along(const Slope& r, float z, float k, float m) {
  const float d = (z - m) * k, p = fast_exp2(d);
  if constexpr (kEntropy) return p * fmaf(r.beta, fmaxf(d, kFloor), r.alpha);
  return p * r.alpha;
}

}  // namespace
}  // namespace pico
