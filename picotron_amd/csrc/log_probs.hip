// Log-probabilities of given tokens from their logits, their gradient, and the two losses made of them: the clipped policy loss
// with a KL term and the preference loss over pairs of answers.  One workgroup per token row, fp32 arithmetic on bf16 or fp32
// logits.  Rows whose target equals ignore_index, or lies outside [0, vocab), where no load may follow, are not read: their
// results are 0 and so is their gradient.
#include <type_traits>
#include "log_probs.h"

namespace pico {
namespace {

constexpr int kUnroll = 4;   // pieces of a row that a thread requests before it uses the first

__device__ __forceinline__ bool is_token(int64_t t, int64_t ignore_index, int vocab) { return t != ignore_index && t >= 0 && t < vocab; }

// (32-bit offsets from the row's address, which is the same for all lanes: a register per access instead of two)
// kKeep: what is loaded is to stay in the caches, to be read again; otherwise it passes them.
template <bool kKeep = false, typename T>
__device__ __forceinline__ u32x4 load_piece(const T* body, uint32_t v) {
  const u32x4* at = reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(body) + v * 16u);
  if constexpr (kKeep) return *at;
  else return __builtin_nontemporal_load(at);
}
template <typename T>
__device__ __forceinline__ void store_piece(T* body, uint32_t v, const float (&e)[io<T>::kVec]) {
  io<T>::store_stream(reinterpret_cast<char*>(body) + v * 16u, e);
}
template <typename T>
__device__ __forceinline__ void unpack(const u32x4& raw, float (&out)[io<T>::kVec]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[2 * i] = __uint_as_float(raw[i] << 16);
      out[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = __uint_as_float(raw[i]);
  }
}

// fn(piece's elements, its index) for every piece of a row that this thread has, NT apart; before(pieces as they were loaded, the first one's index) for kUnroll of
// them at a time
template <typename T, int NT, bool kKeep, typename Fn, typename Before>
__device__ __forceinline__ void each_piece(const Row<T>& r, const Fn& fn, const Before& before) {
  constexpr int V = Row<T>::V, U = kUnroll;
  int v = r.template first<NT>();
  for (int whole = r.nvec / (U * NT); whole > 0; --whole, v += U * NT) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_piece<kKeep>(r.body, v + u * NT);
    before(raw, v);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float e[V];
      unpack<T>(raw[u], e);
      fn(e, v + u * NT);
    }
  }
  // the last ones, requested together too ([1, 64, 32000] 6.5 -> 5.7 us, [16, 1024, 2000] 16.1 -> 12.0)
  u32x4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (v + u * NT < r.nvec) raw[u] = load_piece<kKeep>(r.body, v + u * NT);
  before(raw, v);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (v + u * NT < r.nvec) {
      float e[V];
      unpack<T>(raw[u], e);
      fn(e, v + u * NT);
    }
}

// where a column lies among a row's pieces (piece -1: in the head; one past the last: in the tail)
template <typename T>
struct Place {
  int piece, elem;
  __device__ __forceinline__ Place(const Row<T>& r, int t) : piece(t >= r.head ? (t - r.head) / Row<T>::V : -1), elem(t >= r.head ? (t - r.head) % Row<T>::V : 0) {}
  __device__ __forceinline__ void mask(u32x4& raw) const {   // -inf there, in a piece as it was loaded
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) raw[i] = i == elem ? 0xff800000u : raw[i];
      else raw[i] = i != elem / 2 ? raw[i] : elem % 2 ? (raw[i] & 0xffffu) | 0xff800000u : (raw[i] & 0xffff0000u) | 0xff80u;
    }
  }
  __device__ __forceinline__ void add(float (&e)[Row<T>::V], float v) const {
#pragma unroll
    for (int i = 0; i < Row<T>::V; ++i) e[i] += i == elem ? v : 0.f;
  }
};

template <typename T, int NT, bool kEntropy>
__device__ __forceinline__ Gather<kEntropy> gather_row(const Row<T>& r, int t, float k, bool keep, float (*share)[3]) {   // all but the target
  Gather<kEntropy> g;
  const Place<T> target(r, t);
  const int mine = (target.piece - r.template first<NT>()) % NT == 0 ? target.piece : -1;   // (looked for once in four pieces, by one thread)
  auto add = [&](const float (&e)[Row<T>::V], int) { g.add(e, k); };
  auto without_target = [&](u32x4 (&raw)[kUnroll], int v) {
    if (mine >= v && mine < v + kUnroll * NT) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (mine == v + u * NT) target.mask(raw[u]);
    }
  };
  if (keep) each_piece<T, NT, true>(r, add, without_target);
  else each_piece<T, NT, false>(r, add, without_target);
  if (r.edge >= 0 && r.edge != t) {
    const float e[1] = {static_cast<float>(r.x[r.edge])};
    g.add(e, k);
  }
  join<NT>(g, k, share);
  return g;
}

// the gradient of a row at d; d and r.x lie alike modulo 16 bytes
template <typename T, int NT, bool kEntropy>
__device__ __forceinline__ void write_gradient(const Row<T>& r, T* d, const Slope& slope, float k, float m, int t, bool kept) {
  constexpr int V = Row<T>::V;
  T* body = d + r.head;
  const Place<T> target(r, t);
  auto write = [&](const float (&e)[V], int v) {
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = along<kEntropy>(slope, e[i], k, m);
    if (v == target.piece) target.add(o, slope.hot);
    store_piece(body, v, o);
  };
  auto nothing = [](u32x4 (&)[kUnroll], int) {};
  if (kept) each_piece<T, NT, true>(r, write, nothing);
  else each_piece<T, NT, false>(r, write, nothing);
  if (r.edge >= 0)
    d[r.edge] = static_cast<T>(along<kEntropy>(slope, static_cast<float>(r.x[r.edge]), k, m) + (r.edge == t ? slope.hot : 0.f));
}
template <typename T, int NT>
__device__ __forceinline__ void write_zeros(const Row<T>& r, T* d) {
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int v = r.template first<NT>(); v < r.nvec; v += NT) __builtin_nontemporal_store(zero, reinterpret_cast<u32x4*>(reinterpret_cast<char*>(d + r.head) + static_cast<uint32_t>(v) * 16u));
  if (r.edge >= 0) d[r.edge] = static_cast<T>(0.f);
}

// ---- log-probabilities: one read of the logits
// log_probs, entropy [rows]; max_sum [rows, 2]: what the gradient needs of a row (the maximum and the sum)
template <typename T, int NT, bool kEntropy>
__global__ __launch_bounds__(NT) void log_probs_kernel(const LogitsArgs z, const TokenArgs targets, float* __restrict__ log_probs,
                                                       float* __restrict__ entropy, f32x2* __restrict__ max_sum, int64_t kept_from, int64_t ignore_index) {
  __shared__ float share[NT / kWave][3];
  const int64_t row = blockIdx.x, b = row / z.seq, s = row - b * z.seq;
  const int64_t t = targets.at(b, s);
  if (!is_token(t, ignore_index, z.vocab)) {
    if (threadIdx.x == 0) {
      log_probs[row] = 0.f;
      if constexpr (kEntropy) entropy[row] = 0.f;
      if (max_sum != nullptr) max_sum[row] = f32x2{0.f, 1.f};
    }
    return;
  }
  const Row<T> r(z.data, b * z.batch_stride + s * z.row_stride, z.vocab);
  const float xt = static_cast<float>(r.x[t]);
  Gather<kEntropy> g = gather_row<T, NT, kEntropy>(r, static_cast<int>(t), z.k, row >= kept_from, share);
  if (threadIdx.x == 0) {
    log_probs[row] = with_target(g, xt, z.k, z.inv_t);
    if constexpr (kEntropy) entropy[row] = logf(g.s) - kLn2 * g.w / g.s;
    if (max_sum != nullptr) max_sum[row] = f32x2{g.m, g.s};
  }
}

// ---- their gradient: one read, one write.  d = up (dlp d log p_t + dh dH); up: a device scalar or NULL (1).
// The rows are walked from the last to the first: a loss is usually differentiated as soon as it is there, and what the forward read last lies
// in the 256 MB behind the L2s.  The forward reads the rows from kept_from on such that they stay there, the others past the caches; dlogits leaves
// past them too, or it would push the rows out.  Forward and backward, us: [4, 1024, 49152] bf16 187 -> 173, [3, 777, 32001] fp32 146 -> 132 (128 MB
// kept 178 and 137, 256 MB 174 and 130, but the forward alone 58 instead of 52), [14, 333, 32001] bf16 142 -> 131; everything kept and stores that stay 205,
// 158 and 154.
template <typename T, int NT, bool kEntropy>
__global__ __launch_bounds__(NT) void log_probs_grad_kernel(const LogitsArgs z, const TokenArgs targets, const f32x2* __restrict__ max_sum,
                                                            const float* __restrict__ entropy, const ValueArgs dlp, const ValueArgs dh,
                                                            const float* __restrict__ upstream, int skip_unit, T* __restrict__ dlogits,
                                                            int64_t dbatch_stride, int64_t drow_stride, int64_t rows, int64_t kept_from,
                                                            int64_t ignore_index) {
  const float up = upstream != nullptr ? *upstream : 1.f;
  if (skip_unit && up == 1.f) return;   // dlogits holds the gradient for a unit upstream gradient already
  for (int64_t row = rows - 1 - blockIdx.x; row >= 0; row -= gridDim.x) {
    const int64_t b = row / z.seq, s = row - b * z.seq;
    const int64_t t = targets.at(b, s);
    const Row<T> r(z.data, b * z.batch_stride + s * z.row_stride, z.vocab);
    T* d = dlogits + b * dbatch_stride + s * drow_stride;
    float a = 0.f, h = 0.f;
    if (is_token(t, ignore_index, z.vocab)) {
      if (dlp.data != nullptr) a = dlp.at(b, s) * up;
      if constexpr (kEntropy) h = dh.at(b, s) * up;
    }
    if (a == 0.f && h == 0.f) {   // nothing of the row is needed
      write_zeros<T, NT>(r, d);
      continue;
    }
    const f32x2 ms = max_sum[row];
    write_gradient<T, NT, kEntropy>(r, d, slope<kEntropy>(a, h, ms[1], kEntropy ? entropy[row] : 0.f, z.inv_t), z.k, ms[0], static_cast<int>(t), row >= kept_from);
  }
}

// ---- policy loss.  With q = log p_t (the policy's), A the advantage, old and ref the log-probabilities of the sampling and of the
// reference policy: ratio = exp(q - old), l = -min(ratio A, clamp(ratio, 1 - low, 1 + high) A) + c_kl (exp(ref - q) - (ref - q) - 1)
// - c_h H;  dl/dq = -ratio A where the first is the smaller (and where both are equal) + c_kl (1 - exp(ref - q)),  dl/dH = -c_h.
// A row's gradient depends on the row alone, so loss and gradient are one pass.
struct PolicyArgs {
  ValueArgs advantages, old_lp, ref_lp, weights;   // data NULL: q itself, no KL term, 1 / rows that count
  float low, high, kl_coef, entropy_coef, scale;
  const float* inv_count;   // scale / rows that count, where weights are not given
  float *log_probs, *losses, *dlp, *dentropy, *entropy;   // [rows]; the last three (gradient) or entropy alone may be NULL
  f32x2* max_sum;
};
struct PolicyRow {
  float loss, a, b;   // weighted
};
struct PolicyInputs {   // of a row, requested with its logits
  float A, old, ref, w;
  __device__ __forceinline__ PolicyInputs(const PolicyArgs& p, int64_t b, int64_t s, bool counted) {
    A = p.advantages.at(b, s);
    old = p.old_lp.data != nullptr ? p.old_lp.at(b, s) : 0.f;
    ref = p.ref_lp.data != nullptr ? p.ref_lp.at(b, s) : 0.f;
    w = p.weights.data != nullptr ? p.weights.at(b, s) * p.scale : counted ? *p.inv_count : 1.f;
  }
};
// exp(d) - 1 and exp(d) - 1 - d, which near 0 are sums of what exp(d) has rounded away (a policy next to its reference: of d = 1e-3 the second would be 5 % off, of 1e-4 three times
// itself or negative).  There as a series, whose next term is under 2^-24 of the second.
struct Growth {
  float by, past_line;
  __device__ __forceinline__ explicit Growth(float d) {
    if (fabsf(d) < 0.5f) {
      const float tail = fmaf(d, fmaf(d, fmaf(d, fmaf(d, fmaf(d, 1.f / 40320.f, 1.f / 5040.f), 1.f / 720.f), 1.f / 120.f), 1.f / 24.f), 1.f / 6.f);
      past_line = d * d * fmaf(d, tail, 0.5f);
      by = d + past_line;
    } else {
      by = fast_exp2(d * kLog2e) - 1.f;
      past_line = by - d;
    }
  }
};
__device__ __forceinline__ PolicyRow policy_row(const PolicyArgs& p, const PolicyInputs& in, float q, float H) {
  const float A = in.A, w = in.w;
  const float ratio = p.old_lp.data != nullptr ? fast_exp2((q - in.old) * kLog2e) : q != q ? q : 1.f;   // (no finite loss beside a gradient of NaN)
  const float held = fminf(fmaxf(ratio, p.low), p.high), free = ratio * A, bound = held * A;
  PolicyRow r;
  // (written such that a NaN anywhere comes out)
  r.loss = bound < free ? -bound : -free;
  r.a = bound < free ? 0.f : -free;
  if (p.ref_lp.data != nullptr && p.kl_coef != 0.f) {
    const Growth grow(in.ref - q);
    r.loss += p.kl_coef * grow.past_line;
    r.a -= p.kl_coef * grow.by;
  }
  r.b = 0.f;
  if (p.entropy_coef != 0.f) {
    r.loss -= p.entropy_coef * H;
    r.b = -p.entropy_coef * w;
  }
  r.loss *= w;
  r.a *= w;
  return r;
}

template <typename T, int NT, bool kEntropy, bool kGrad>
__global__ __launch_bounds__(NT) void policy_kernel(const LogitsArgs z, const TokenArgs targets, const PolicyArgs p, T* __restrict__ dlogits,
                                                    int64_t dbatch_stride, int64_t drow_stride, int64_t ignore_index) {
  __shared__ float share[NT / kWave][3];
  const int64_t row = blockIdx.x, b = row / z.seq, s = row - b * z.seq;
  const int64_t t = targets.at(b, s);
  const Row<T> r(z.data, b * z.batch_stride + s * z.row_stride, z.vocab);
  T* d = kGrad ? dlogits + b * dbatch_stride + s * drow_stride : nullptr;
  if (!is_token(t, ignore_index, z.vocab)) {
    if constexpr (kGrad) write_zeros<T, NT>(r, d);
    if (threadIdx.x == 0) {
      p.log_probs[row] = p.losses[row] = 0.f;
      if constexpr (kGrad) {
        p.dlp[row] = 0.f;
        if constexpr (kEntropy) p.dentropy[row] = p.entropy[row] = 0.f;
        p.max_sum[row] = f32x2{0.f, 1.f};
      }
    }
    return;
  }
  const float xt = static_cast<float>(r.x[t]);
  const PolicyInputs in(p, b, s, kGrad);
  Gather<kEntropy> g = gather_row<T, NT, kEntropy>(r, static_cast<int>(t), z.k, kGrad, share);   // (with a gradient the row is read again below)
  float q = with_target(g, xt, z.k, z.inv_t);
  asm volatile("" : "+v"(q));   // (rounded as it is stored, or its difference from `old` is taken before the rounding: where they are equal the ratio is 1)
  const float H = kEntropy ? logf(g.s) - kLn2 * g.w / g.s : 0.f;
  const PolicyRow l = policy_row(p, in, q, H);
  if (threadIdx.x == 0) {
    p.log_probs[row] = q;
    p.losses[row] = l.loss;
    if constexpr (kGrad) {
      p.dlp[row] = l.a;
      if constexpr (kEntropy) { p.dentropy[row] = l.b; p.entropy[row] = H; }
      p.max_sum[row] = f32x2{g.m, g.s};
    }
  }
  if constexpr (kGrad) write_gradient<T, NT, kEntropy>(r, d, slope<kEntropy>(l.a, l.b, g.s, H, z.inv_t), z.k, g.m, static_cast<int>(t), true);
}

// The same with the row in registers between its statistics and its gradient: the logits are read once.  NT threads hold NV pieces of 16 bytes each, packed as
// they came; each phase unpacks them again (the empty asm hides that it is the same value, or the compiler would keep the unpacked row).
// count_rows > 0 (at most NT; targets without gaps): every workgroup counts the rows that count for itself, behind the requests for its row, instead of a
// launch in front.
template <typename T, int NT, int NV, bool kEntropy>
__global__ __launch_bounds__(NT, NV <= 6 ? 8 : NV <= 8 ? 6 : NV <= 12 ? 5 : 4) void policy_held_kernel(const LogitsArgs z, const TokenArgs targets, const PolicyArgs p, T* __restrict__ dlogits,
                                                                         int64_t dbatch_stride, int64_t drow_stride, int64_t ignore_index, int count_rows) {
  constexpr int V = Row<T>::V, W = NT / kWave;
  __shared__ float share[W][3];
  __shared__ int counted[W];
  const int64_t row = blockIdx.x, b = row / z.seq, s = row - b * z.seq;
  const int64_t t = targets.at(b, s);
  const Row<T> r(z.data, b * z.batch_stride + s * z.row_stride, z.vocab);
  T* d = dlogits + b * dbatch_stride + s * drow_stride;
  if (!is_token(t, ignore_index, z.vocab)) {
    write_zeros<T, NT>(r, d);
    if (threadIdx.x == 0) {
      p.log_probs[row] = p.losses[row] = p.dlp[row] = 0.f;
      if constexpr (kEntropy) p.dentropy[row] = p.entropy[row] = 0.f;
      p.max_sum[row] = f32x2{0.f, 1.f};
    }
    return;
  }
  constexpr uint32_t kNegInf = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;   // past the end of the row: its exponential is 0
  const int first = r.template first<NT>();
  u32x4 raw[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = first + j * NT;
    raw[j] = u32x4{kNegInf, kNegInf, kNegInf, kNegInf};
    if (v < r.nvec) raw[j] = load_piece(r.body, v);
  }
  auto hide = [&]() {
#pragma unroll
    for (int j = 0; j < NV; ++j) asm volatile("" : "+v"(raw[j]));
  };
  const float xt = static_cast<float>(r.x[t]), xe = r.edge >= 0 ? static_cast<float>(r.x[r.edge]) : -INFINITY;
  PolicyInputs in(p, b, s, count_rows == 0);
  if (count_rows > 0) {
    const int64_t other = static_cast<int>(threadIdx.x) < count_rows ? targets.data[threadIdx.x] : ignore_index;
    const int n = __popcll(__ballot(is_token(other, ignore_index, z.vocab)));
    if (threadIdx.x % kWave == 0) counted[threadIdx.x / kWave] = n;
    if constexpr (W == 1) __syncthreads();   // (otherwise the one in join)
  }
  Gather<kEntropy> g;
  float top = xe;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float e[V];
    unpack<T>(raw[j], e);
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, e[i]);
  }
  g.rise(top, z.k);
  const int ti = static_cast<int>(t);
  const Place<T> target(r, ti);
  hide();
  {
    const float e[1] = {xe};
    g.take(e, z.k);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float e[V];
    unpack<T>(raw[j], e);
    g.take(e, z.k);
    __builtin_amdgcn_sched_barrier(0);
  }
  hide();
  join<NT>(g, z.k, share);
  if (count_rows > 0) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) n += counted[i];
    in.w = p.scale / static_cast<float>(n);   // (this row is one of them)
  }
  float q = (xt - g.zmax) * z.inv_t - logf(g.s);   // (the target among the others: taking it out of a row that is held costs registers that are not there)
  asm volatile("" : "+v"(q));   // (rounded as it is stored, or its difference from `old` is taken before the rounding: where they are equal the ratio is 1)
  const float H = kEntropy ? logf(g.s) - kLn2 * g.w / g.s : 0.f;
  const PolicyRow l = policy_row(p, in, q, H);
  if (threadIdx.x == 0) {
    p.log_probs[row] = q;
    p.losses[row] = l.loss;
    p.dlp[row] = l.a;
    if constexpr (kEntropy) { p.dentropy[row] = l.b; p.entropy[row] = H; }
    p.max_sum[row] = f32x2{g.m, g.s};
  }
  const Slope along_row = slope<kEntropy>(l.a, l.b, g.s, H, z.inv_t);
  T* body = d + r.head;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = first + j * NT;
    if (v < r.nvec) {
      float e[V];
      unpack<T>(raw[j], e);
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = along<kEntropy>(along_row, e[i], z.k, g.m);
      if (v == target.piece) target.add(e, along_row.hot);
      store_piece(body, v, e);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if (r.edge >= 0) d[r.edge] = static_cast<T>(along<kEntropy>(along_row, xe, z.k, g.m) + (r.edge == ti ? along_row.hot : 0.f));
}

// ---- sums over rows: one workgroup, in double and in a fixed order
constexpr int kSumThreads = 1024, kSumWaves = kSumThreads / kWave;
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

// count: inv_count = scale / max(rows that count, 1); with `loss`: the sum of the losses, times that where they are not weighted yet, and so are they then
__global__ __launch_bounds__(kSumThreads) void policy_sum_kernel(const TokenArgs targets, float* __restrict__ losses, float* __restrict__ loss,
                                                                 float* __restrict__ inv_count, float scale, int count, int unweighted,
                                                                 int64_t rows, int seq, int vocab, int64_t ignore_index) {
  __shared__ double red_s[kSumWaves];
  __shared__ int red_n[kSumWaves];
  __shared__ float factor;
  double sum = 0;
  int n = 0;
  constexpr int U = 8;   // rows requested together
  for (int64_t first = threadIdx.x; first < rows; first += U * kSumThreads) {
    float l[U];
    int64_t t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = first + u * kSumThreads, b = row / seq;
      const bool in = row < rows;
      t[u] = in && count ? targets.at(b, row - b * seq) : ignore_index;
      l[u] = in && loss != nullptr ? losses[row] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      n += is_token(t[u], ignore_index, vocab);
      sum += l[u];
    }
  }
  sum = wave_sum64(sum);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, kWave);
  if (threadIdx.x % kWave == 0) { red_s[threadIdx.x / kWave] = sum; red_n[threadIdx.x / kWave] = n; }
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0;
    int all = 0;
    for (int w = 0; w < kSumWaves; ++w) { total += red_s[w]; all += red_n[w]; }
    const float inv = scale / static_cast<float>(all > 0 ? all : 1);
    if (count) *inv_count = inv;
    if (loss != nullptr) *loss = static_cast<float>(unweighted ? total * inv : total);
    factor = inv;
  }
  if (loss == nullptr || !unweighted) return;
  __syncthreads();
  const float by = factor;
  for (int64_t first = threadIdx.x; first < rows; first += U * kSumThreads) {
    float l[U];
#pragma unroll
    for (int u = 0; u < U; ++u) l[u] = first + u * kSumThreads < rows ? losses[first + u * kSumThreads] : 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + u * kSumThreads < rows) losses[first + u * kSumThreads] = l[u] * by;
  }
}

// ---- preference loss over pairs: sequences i (chosen) and pairs + i (rejected).  L = sum or mean of the log-probabilities of a
// sequence's tokens that count; x = beta ((L_c - ref_c) - (L_r - ref_r));  l = (1 - e) softplus(-x) + e softplus(x);
// dl/dx = -(1 - e) sigmoid(-x) + e sigmoid(x).  Sums of thousands of log-probabilities from which a reference's nearly equal sum is
// taken: in double.  One workgroup; the waves of a team share a sequence.
struct PreferenceArgs {
  const float *log_probs, *ref;   // [rows]; [2 pairs] or NULL
  float *loss, *sequence, *slope; // [1]; [2 pairs] L; [2 pairs]: dloss / d log p of each of the sequence's tokens
  double* sums;                   // [2 pairs]
  float beta, smoothing, scale;
  int average;
};
__global__ __launch_bounds__(kSumThreads) void preference_kernel(const TokenArgs targets, const PreferenceArgs p, int pairs, int seq, int vocab,
                                                                 int64_t ignore_index) {
  __shared__ double red_s[kSumWaves];
  __shared__ int red_n[kSumWaves];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, sequences = 2 * pairs;
  int team = 1;   // waves
  while (team < kSumWaves && sequences * team * 2 <= kSumWaves) team *= 2;
  const int teams = kSumWaves / team;
  for (int first = 0; first < sequences; first += teams) {
    const int b = first + wave / team;
    double sum = 0;
    int n = 0;
    if (b < sequences) {
      constexpr int U = 4;   // tokens requested together
      const int step = team * kWave;
      for (int64_t first = wave % team * kWave + lane; first < seq; first += U * step) {
        float q[U];
        int64_t t[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t s = first + u * step;
          q[u] = s < seq ? p.log_probs[static_cast<int64_t>(b) * seq + s] : 0.f;
          t[u] = s < seq && p.average ? targets.at(b, s) : ignore_index;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          sum += q[u];
          n += is_token(t[u], ignore_index, vocab);
        }
      }
    }
    sum = wave_sum64(sum);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, kWave);
    if (lane == 0) { red_s[wave] = sum; red_n[wave] = n; }
    __syncthreads();
    if (wave % team == 0 && lane == 0 && b < sequences) {
      for (int w = 1; w < team; ++w) { sum += red_s[wave + w]; n += red_n[wave + w]; }
      const double over = p.average && n > 0 ? n : 1;
      p.sums[b] = sum / over;
      p.sequence[b] = static_cast<float>(sum / over);
      p.slope[b] = static_cast<float>(1 / over);   // (for the pair's factor below)
    }
    __syncthreads();
  }
  __threadfence_block();
  __syncthreads();
  double loss = 0;
  for (int i = threadIdx.x; i < pairs; i += kSumThreads) {
    double x = p.sums[i] - p.sums[pairs + i];
    if (p.ref != nullptr) x -= static_cast<double>(p.ref[i]) - static_cast<double>(p.ref[pairs + i]);
    x *= p.beta;
    const double e = p.smoothing, small = exp(-fabs(x)), part = log1p(small);   // softplus(x) = max(x, 0) + log(1 + exp(-|x|))
    loss += (e < 1 ? (1 - e) * (fmax(-x, 0.) + part) : 0.) + (e > 0 ? e * (fmax(x, 0.) + part) : 0.);
    const double up = (x > 0 ? 1. : small) / (1 + small), down = (x > 0 ? small : 1.) / (1 + small);   // sigmoid(x), sigmoid(-x)
    const double dx = (e * up - (1 - e) * down) * p.beta * p.scale / pairs;
    p.slope[i] = static_cast<float>(dx * p.slope[i]);
    p.slope[pairs + i] = static_cast<float>(-dx * p.slope[pairs + i]);
  }
  loss = wave_sum64(loss);
  if (lane == 0) red_s[wave] = loss;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0;
    for (int w = 0; w < kSumWaves; ++w) total += red_s[w];
    *p.loss = static_cast<float>(total * p.scale / (pairs > 0 ? pairs : 1));
  }
}

// ---- launches
template <int n> using Int = std::integral_constant<int, n>;
// the narrowest workgroup that has a row in four pieces a thread, eight from 256 threads on: in a wider one most lanes of a short row would idle.
// Long rows of the gradient in 1024: [4, 1024, 49152] bf16 124 -> 120 us ([14, 333, 32001], 4000 pieces, 79 -> 92; the forward 52 -> 56).
template <bool kGrad, typename Fn>
void with_threads(int64_t vocab, int vec, const Fn& fn) {
  const int64_t pieces = (vocab + vec - 1) / vec;
  if (pieces <= 64 * 4) fn(Int<64>());
  else if (pieces <= 128 * 4) fn(Int<128>());
  else if (pieces <= 256 * 8) fn(Int<256>());
  else if (!kGrad || pieces < 1024 * 5) fn(Int<512>());
  else if constexpr (kGrad) fn(Int<1024>());
}
// Threads and pieces per thread of the kernel that holds a row of so many pieces; (0, 0): none does.  As few threads as can hold the row in four or eight pieces: a
// barrier over fewer waves, and more rows on a CU.  6144 pieces in 1024 x 6, where two rows share a CU, [8, 1024, 49152] bf16 256 us, in 512 x 12 262; with an entropy
// term the former has no registers left (12 bytes of scratch).  The long rows, us of 400 MB of logits (a copy: 162), without and with an entropy term, held here, in 1024
// threads up to 8192 pieces (12288 for the last rung), and read twice:
//   bf16  49160   147, 159 | 180, 195 | 181, 182      bf16 131072   160, 173 |    -     | 187, 189
//   bf16  65536   151, 156 | 162, 176 | 179, 180      fp32  25000   144, 143 | 149, 157 | 179, 180
//   bf16  65544   188, 221 | 187, 201 | 179, 180      fp32  32772   155, 161 | 160, 164 | 178, 179
//   bf16  80000   179, 201 | 180, 191 | 180, 181      fp32  50000   152, 156 |    -     | 182, 183
//   bf16 100000   168, 190 |    -     | 182, 185      fp32  65536   152, 152 |    -     | 182, 183
// (1024 x 16 leaves one row on a CU, whose phases nothing overlaps: just past 8192 pieces of bf16 it loses 5 to 23 %.  Past 16384, read twice, 131080 bf16 187, 190, 128256 fp32
// 227, 230.)
template <bool kEntropy, typename Fn>
void with_pieces(int64_t vocab, int vec, const Fn& fn) {
  const int64_t pieces = vocab / vec;
  if (pieces <= 64 * 4) fn(Int<64>(), Int<4>());
  else if (pieces <= 128 * 4) fn(Int<128>(), Int<4>());
  else if (pieces <= 256 * 4) fn(Int<256>(), Int<4>());
  else if (pieces <= 256 * 8) fn(Int<256>(), Int<8>());
  else if (pieces <= 512 * 8) fn(Int<512>(), Int<8>());
  else if (pieces <= 1024 * 6) {
    if constexpr (kEntropy) fn(Int<512>(), Int<12>());
    else fn(Int<1024>(), Int<6>());
  } else if (pieces <= 512 * 16) fn(Int<512>(), Int<16>());
  else if (pieces <= 1024 * 16) fn(Int<1024>(), Int<16>());
  else fn(Int<0>(), Int<0>());
}
template <bool kGrad, typename Fn>
void with_type(const pico_logits& z, const Fn& fn) {
  if (z.dtype == PICO_BF16) with_threads<kGrad>(z.vocab, 8, [&](auto nt) { fn(__bf16(), nt); });
  else with_threads<kGrad>(z.vocab, 4, [&](auto nt) { fn(float(), nt); });
}
template <typename Fn>
void with_flag(bool v, const Fn& fn) {
  if (v) fn(std::true_type());
  else fn(std::false_type());
}

int check_logits(const char* fn, const pico_logits* z, const pico_tokens* targets, float temperature) {
  if (!z || !targets) return fail(PICO_ERR_NULL, "%s: logits and targets are required", fn);
  if (z->dtype != PICO_BF16 && z->dtype != PICO_F32) return fail(PICO_ERR_DTYPE, "%s: dtype code %d not supported", fn, z->dtype);
  constexpr int64_t kMost = 0x7fffffff;
  // (one workgroup per row; vocab: a row's index fits 32 bits with room for the pieces of an unrolled step)
  if (z->batch < 0 || z->seq < 0 || z->vocab <= 0 || z->vocab > kMost / 4 || z->seq > kMost || z->batch > kMost || z->batch * z->seq > kMost)
    return fail(PICO_ERR_SHAPE, "%s: batch=%lld seq=%lld vocab=%lld", fn, static_cast<long long>(z->batch), static_cast<long long>(z->seq),
                static_cast<long long>(z->vocab));
  // (a launch has fewer than 2^32 threads)
  const int64_t threads = z->vocab <= 2048 ? 128 : z->vocab <= 8192 ? 256 : 1024;
  if (z->batch * z->seq > 0xffffffffll / threads)
    return fail(PICO_ERR_SHAPE, "%s: %lld rows of %lld, at most %lld", fn, static_cast<long long>(z->batch * z->seq), static_cast<long long>(z->vocab), 0xffffffffll / threads);
  if (!(temperature > 0.f) || !(temperature <= 1e30f) || !(1.f / temperature <= 1e30f)) return fail(PICO_ERR_SHAPE, "%s: temperature %g must be positive and finite", fn, temperature);
  if (z->batch * z->seq > 0) {
    if (!z->data || !targets->data) return fail(PICO_ERR_NULL, "%s: logits and targets are required", fn);
    const int size = z->dtype == PICO_BF16 ? 2 : 4;
    if (reinterpret_cast<uintptr_t>(z->data) % size) return fail(PICO_ERR_ALIGN, "%s: logits must be aligned to their elements", fn);
    if (z->batch_stride < 0 || z->row_stride < 0) return fail(PICO_ERR_STRIDE, "%s: strides of the logits must not be negative", fn);
  }
  return PICO_OK;
}
// dlogits: rows of their own, each as far from a 16-byte boundary as the row of logits
int check_gradient(const char* fn, const pico_logits& z, const void* d, int64_t dbatch_stride, int64_t drow_stride) {
  const int64_t vec = z.dtype == PICO_BF16 ? 8 : 4;
  if ((z.seq > 1 && drow_stride < z.vocab) || (z.batch > 1 && dbatch_stride < (z.seq - 1) * drow_stride + z.vocab))
    return fail(PICO_ERR_STRIDE, "%s: the rows of dlogits overlap", fn);
  if ((reinterpret_cast<uintptr_t>(z.data) - reinterpret_cast<uintptr_t>(d)) % 16 != 0 || (z.seq > 1 && (drow_stride - z.row_stride) % vec != 0) ||
      (z.batch > 1 && (dbatch_stride - z.batch_stride) % vec != 0))
    return fail(PICO_ERR_ALIGN, "%s: a row of dlogits has to lie as far from a 16-byte boundary as its row of logits", fn);
  return PICO_OK;
}
LogitsArgs args(const pico_logits& z, float temperature) {
  const float inv_t = 1.f / temperature;
  return {z.data, z.batch_stride, z.row_stride, static_cast<int>(z.seq), static_cast<int>(z.vocab), static_cast<float>(1.4426950408889634 / temperature), inv_t};
}
// the first row that the forward keeps in the caches for the backward
constexpr int64_t kKeptBytes = int64_t{160} << 20;
int64_t kept_from(const pico_logits& z) {
  const int64_t rows = z.batch * z.seq, most = kKeptBytes / (z.vocab * (z.dtype == PICO_BF16 ? 2 : 4));
  return std::max<int64_t>(rows - most, 0);
}
TokenArgs args(const pico_tokens& t) { return {t.data, t.batch_stride, t.row_stride}; }
ValueArgs args(const pico_values* v) { return v ? ValueArgs{v->data, v->batch_stride, v->row_stride} : ValueArgs{nullptr, 0, 0}; }

int run_log_probs(const char* fn, const pico_logits& z, const pico_tokens& targets, float* log_probs, float* entropy, float* max_sum,
                  float temperature, int64_t ignore_index, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(z.batch * z.seq));
  with_type<false>(z, [&](auto type, auto nt) {
    with_flag(entropy != nullptr, [&](auto with) {
      hipLaunchKernelGGL((log_probs_kernel<decltype(type), decltype(nt)::value, decltype(with)::value>), grid, dim3(decltype(nt)::value), 0, s, args(z, temperature),
                         args(targets), log_probs, entropy, reinterpret_cast<f32x2*>(max_sum), max_sum ? kept_from(z) : z.batch * z.seq, ignore_index);
    });
  });
  return check_launch(fn);
}

}  // namespace
}  // namespace pico

using namespace pico;

extern "C" int pico_log_probs_fwd(const pico_logits* logits, const pico_tokens* targets, float* log_probs, float* entropy, float* max_sum,
                                  float temperature, int64_t ignore_index, void* stream) {
  const char* fn = "pico_log_probs_fwd";
  if (int rc = check_logits(fn, logits, targets, temperature)) return rc;
  if (logits->batch * logits->seq == 0) return PICO_OK;
  if (!log_probs) return fail(PICO_ERR_NULL, "%s: log_probs is required", fn);
  if (reinterpret_cast<uintptr_t>(max_sum) % 8) return fail(PICO_ERR_ALIGN, "%s: max_sum must be aligned to 8 bytes", fn);
  return run_log_probs(fn, *logits, *targets, log_probs, entropy, max_sum, temperature, ignore_index, static_cast<hipStream_t>(stream));
}

extern "C" int pico_log_probs_bwd(const pico_logits* logits, const pico_tokens* targets, const float* max_sum, const float* entropy,
                                  const pico_values* dlog_probs, const pico_values* dentropy, const float* grad_out, int have_unit,
                                  void* dlogits, int64_t dbatch_stride, int64_t drow_stride, float temperature, int64_t ignore_index, void* stream) {
  const char* fn = "pico_log_probs_bwd";
  if (int rc = check_logits(fn, logits, targets, temperature)) return rc;
  const int64_t rows = logits->batch * logits->seq;
  if (rows == 0) return PICO_OK;
  const bool with_entropy = dentropy && dentropy->data;
  if (!max_sum || !dlogits || (!with_entropy && !(dlog_probs && dlog_probs->data)) || (with_entropy && !entropy) || (have_unit && !grad_out))
    return fail(PICO_ERR_NULL, "%s: max_sum, dlogits, one of dlog_probs and dentropy, entropy with the latter and grad_out with have_unit are required", fn);
  if (reinterpret_cast<uintptr_t>(max_sum) % 8) return fail(PICO_ERR_ALIGN, "%s: max_sum must be aligned to 8 bytes", fn);
  if (int rc = check_gradient(fn, *logits, dlogits, dbatch_stride, drow_stride)) return rc;
  // (with the gradient at hand the launch usually only looks at grad_out: as many workgroups as the GPU holds at once, which walk the rows if they must)
  const dim3 grid(static_cast<unsigned>(have_unit ? std::min<int64_t>(rows, 512) : rows));
  with_type<true>(*logits, [&](auto type, auto nt) {
    with_flag(with_entropy, [&](auto with) {
      hipLaunchKernelGGL((log_probs_grad_kernel<decltype(type), decltype(nt)::value, decltype(with)::value>), grid, dim3(decltype(nt)::value), 0, static_cast<hipStream_t>(stream),
                         args(*logits, temperature), args(*targets), reinterpret_cast<const f32x2*>(max_sum), entropy, args(dlog_probs), args(dentropy),
                         grad_out, have_unit, static_cast<decltype(type)*>(dlogits), dbatch_stride, drow_stride, rows, kept_from(*logits), ignore_index);
    });
  });
  return check_launch(fn);
}

extern "C" int pico_policy_loss_fwd(const pico_logits* logits, const pico_tokens* targets, const pico_policy* policy, float* loss, float* log_probs,
                                    float* losses, float* inv_count, const pico_policy_saved* saved, void* dlogits, int64_t dbatch_stride,
                                    int64_t drow_stride, float temperature, int64_t ignore_index, void* stream) {
  const char* fn = "pico_policy_loss_fwd";
  if (int rc = check_logits(fn, logits, targets, temperature)) return rc;
  if (!policy || !loss || !inv_count) return fail(PICO_ERR_NULL, "%s: policy, loss and inv_count are required", fn);
  if (!(policy->clip_low >= 0.f) || !(policy->clip_high >= 0.f)) return fail(PICO_ERR_SHAPE, "%s: clip (%g, %g) must not be negative", fn, policy->clip_low, policy->clip_high);
  const int64_t rows = logits->batch * logits->seq;
  const bool with_entropy = policy->entropy_coef != 0.f, weighted = policy->weights.data != nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows > 0) {
    if (!policy->advantages.data || !log_probs || !losses) return fail(PICO_ERR_NULL, "%s: advantages, log_probs and losses are required", fn);
    if (policy->kl_coef != 0.f && !policy->ref_log_probs.data) return fail(PICO_ERR_NULL, "%s: a KL term needs ref_log_probs", fn);
    if (dlogits) {
      if (!saved || !saved->max_sum || !saved->dlog_probs || (with_entropy && (!saved->entropy || !saved->dentropy)))
        return fail(PICO_ERR_NULL, "%s: with dlogits saved is required, its entropy and dentropy with an entropy term", fn);
      if (reinterpret_cast<uintptr_t>(saved->max_sum) % 8) return fail(PICO_ERR_ALIGN, "%s: max_sum must be aligned to 8 bytes", fn);
      if (int rc = check_gradient(fn, *logits, dlogits, dbatch_stride, drow_stride)) return rc;
    }
  }
  auto sum = [&](float* to) {
    hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(kSumThreads), 0, s, args(*targets), losses, to, inv_count, policy->scale, !weighted && (!to || !dlogits),
                       !weighted && !dlogits, rows, static_cast<int>(std::max<int64_t>(logits->seq, 1)), static_cast<int>(logits->vocab), ignore_index);
  };
  if (rows > 0) {
    PolicyArgs p = {args(&policy->advantages), args(&policy->old_log_probs), args(&policy->ref_log_probs), args(&policy->weights),
                    1.f - policy->clip_low, 1.f + policy->clip_high, policy->kl_coef, policy->entropy_coef, policy->scale, inv_count, log_probs, losses,
                    nullptr, nullptr, nullptr, nullptr};
    if (dlogits) {
      p.dlp = saved->dlog_probs;
      p.dentropy = saved->dentropy;
      p.entropy = saved->entropy;
      p.max_sum = reinterpret_cast<f32x2*>(saved->max_sum);
    }
    const dim3 grid(static_cast<unsigned>(rows));
    auto stream_row = [&](auto type, auto nt, auto with, auto grad) {
      using T = decltype(type);
      constexpr int NT = decltype(nt)::value;
      hipLaunchKernelGGL((policy_kernel<T, NT, decltype(with)::value, decltype(grad)::value>), grid, dim3(NT), 0, s, args(*logits, temperature), args(*targets), p,
                         static_cast<T*>(dlogits), dbatch_stride, drow_stride, ignore_index);
    };
    auto with_gradient = [&](auto type, auto with) {
      using T = decltype(type);
      with_pieces<decltype(with)::value>(logits->vocab, io<T>::kVec, [&](auto nt, auto nv) {
        constexpr int NT = decltype(nt)::value, NV = decltype(nv)::value;
        const bool itself = rows <= NT && targets->row_stride == 1 && (logits->batch == 1 || targets->batch_stride == logits->seq);
        if (!weighted && !itself) sum(nullptr);   // the gradient needs scale / count
        if constexpr (NT == 0) stream_row(type, Int<512>(), with, std::true_type());
        else
          hipLaunchKernelGGL((policy_held_kernel<T, NT, NV, decltype(with)::value>), grid, dim3(NT), 0, s, args(*logits, temperature), args(*targets), p,
                             static_cast<T*>(dlogits), dbatch_stride, drow_stride, ignore_index, !weighted && itself ? static_cast<int>(rows) : 0);
      });
    };
    with_flag(with_entropy, [&](auto with) {
      if (!dlogits) with_type<false>(*logits, [&](auto type, auto nt) { stream_row(type, nt, with, std::false_type()); });
      else if (logits->dtype == PICO_BF16) with_gradient(__bf16(), with);
      else with_gradient(float(), with);
    });
  }
  sum(loss);
  return check_launch(fn);
}

extern "C" int pico_preference_loss_fwd(const pico_logits* logits, const pico_tokens* targets, const float* ref_log_probs, float beta,
                                        float label_smoothing, int average, float scale, float* loss, float* sequence_log_probs, float* slope,
                                        float* log_probs, float* max_sum, void* workspace, int64_t ignore_index, void* stream) {
  const char* fn = "pico_preference_loss_fwd";
  if (int rc = check_logits(fn, logits, targets, 1.f)) return rc;
  if (logits->batch % 2) return fail(PICO_ERR_SHAPE, "%s: batch=%lld must be even (the chosen sequences, then the rejected ones)", fn, static_cast<long long>(logits->batch));
  if (!(label_smoothing >= 0.f && label_smoothing <= 1.f)) return fail(PICO_ERR_SHAPE, "%s: label_smoothing %g must lie in [0, 1]", fn, label_smoothing);
  if (!loss) return fail(PICO_ERR_NULL, "%s: loss is required", fn);
  const int64_t rows = logits->batch * logits->seq;
  if (logits->batch > 0 && (!sequence_log_probs || !slope || !workspace)) return fail(PICO_ERR_NULL, "%s: sequence_log_probs, slope and workspace are required", fn);
  if (rows > 0 && !log_probs) return fail(PICO_ERR_NULL, "%s: log_probs is required", fn);
  if (reinterpret_cast<uintptr_t>(workspace) % 8 || reinterpret_cast<uintptr_t>(max_sum) % 8) return fail(PICO_ERR_ALIGN, "%s: workspace and max_sum must be aligned to 8 bytes", fn);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows > 0)
    if (int rc = run_log_probs(fn, *logits, *targets, log_probs, nullptr, max_sum, 1.f, ignore_index, s)) return rc;
  const PreferenceArgs p = {log_probs, ref_log_probs, loss, sequence_log_probs, slope, static_cast<double*>(workspace), beta, label_smoothing, scale, average};
  hipLaunchKernelGGL(preference_kernel, dim3(1), dim3(kSumThreads), 0, s, args(*targets), p, static_cast<int>(logits->batch / 2), static_cast<int>(logits->seq),
                     static_cast<int>(logits->vocab), ignore_index);
  return check_launch(fn);
}
