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

// fn(piece's elements, its first index) for every piece of a row that this thread has
template <typename T, int NT, typename Fn>
__device__ __forceinline__ void each_piece(const Row<T>& r, const Fn& fn) {
  constexpr int V = Row<T>::V, U = kUnroll;
  int v = threadIdx.x;
  for (; v + (U - 1) * NT < r.nvec; v += U * NT) {
    float e[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) io<T>::load_stream(r.body + static_cast<int64_t>(v + u * NT) * V, e[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) fn(e[u], v + u * NT);
  }
  for (; v < r.nvec; v += NT) {
    float e[V];
    io<T>::load_stream(r.body + static_cast<int64_t>(v) * V, e);
    fn(e, v);
  }
}

template <typename T, int NT, bool kEntropy>
__device__ __forceinline__ Gather<kEntropy> gather_row(const Row<T>& r, float k, float (*share)[3]) {
  Gather<kEntropy> g;
  each_piece<T, NT>(r, [&](const float (&e)[Row<T>::V], int) { g.add(e, k); });
  if (r.edge >= 0) {
    const float e[1] = {static_cast<float>(r.x[r.edge])};
    g.add(e, k);
  }
  join<NT>(g, k, share);
  return g;
}

// the gradient of a row at d; d and r.x lie alike modulo 16 bytes
template <typename T, int NT, bool kEntropy>
__device__ __forceinline__ void write_gradient(const Row<T>& r, T* d, const Slope& slope, float k, float m, int t) {
  constexpr int V = Row<T>::V;
  T* body = d + r.head;
  const int t_piece = t >= r.head ? (t - r.head) / V : -1, t_elem = t >= r.head ? (t - r.head) % V : 0;
  each_piece<T, NT>(r, [&](const float (&e)[V], int v) {
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = along<kEntropy>(slope, e[i], k, m);
    if (v == t_piece) {
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] += i == t_elem ? slope.hot : 0.f;
    }
    io<T>::store_stream(body + static_cast<int64_t>(v) * V, o);
  });
  if (r.edge >= 0)
    d[r.edge] = static_cast<T>(along<kEntropy>(slope, static_cast<float>(r.x[r.edge]), k, m) + (r.edge == t ? slope.hot : 0.f));
}
template <typename T, int NT>
__device__ __forceinline__ void write_zeros(const Row<T>& r, T* d) {
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int v = threadIdx.x; v < r.nvec; v += NT) __builtin_nontemporal_store(zero, reinterpret_cast<u32x4*>(d + r.head + static_cast<int64_t>(v) * Row<T>::V));
  if (r.edge >= 0) d[r.edge] = static_cast<T>(0.f);
}

// ---- log-probabilities: one read of the logits
// log_probs, entropy [rows]; max_sum [rows, 2]: what the gradient needs of a row (the maximum and the sum)
template <typename T, int NT, bool kEntropy>
__global__ __launch_bounds__(NT) void log_probs_kernel(const LogitsArgs z, const TokenArgs targets, float* __restrict__ log_probs,
                                                       float* __restrict__ entropy, f32x2* __restrict__ max_sum, int64_t ignore_index) {
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
  const Gather<kEntropy> g = gather_row<T, NT, kEntropy>(r, z.k, share);
  if (threadIdx.x == 0) {
    log_probs[row] = (xt - g.zmax) * z.inv_t - logf(g.s);
    if constexpr (kEntropy) entropy[row] = logf(g.s) - kLn2 * g.w / g.s;
    if (max_sum != nullptr) max_sum[row] = f32x2{g.m, g.s};
  }
}

// ---- their gradient: one read, one write.  d = up (dlp d log p_t + dh dH); up: a device scalar or NULL (1).
template <typename T, int NT, bool kEntropy>
__global__ __launch_bounds__(NT) void log_probs_grad_kernel(const LogitsArgs z, const TokenArgs targets, const f32x2* __restrict__ max_sum,
                                                            const float* __restrict__ entropy, const ValueArgs dlp, const ValueArgs dh,
                                                            const float* __restrict__ upstream, int skip_unit, T* __restrict__ dlogits,
                                                            int64_t dbatch_stride, int64_t drow_stride, int64_t rows, int64_t ignore_index) {
  const float up = upstream != nullptr ? *upstream : 1.f;
  if (skip_unit && up == 1.f) return;   // dlogits holds the gradient for a unit upstream gradient already
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
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
    write_gradient<T, NT, kEntropy>(r, d, slope<kEntropy>(a, h, ms[1], kEntropy ? entropy[row] : 0.f, z.inv_t), z.k, ms[0], static_cast<int>(t));
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
__device__ __forceinline__ PolicyRow policy_row(const PolicyArgs& p, int64_t b, int64_t s, float q, float H, float w) {
  const float A = p.advantages.at(b, s);
  const float ratio = p.old_lp.data != nullptr ? expf(q - p.old_lp.at(b, s)) : 1.f;
  const float held = fminf(fmaxf(ratio, p.low), p.high), free = ratio * A, bound = held * A;
  PolicyRow r;
  // (written such that a NaN anywhere comes out)
  r.loss = bound < free ? -bound : -free;
  r.a = bound < free ? 0.f : -free;
  if (p.ref_lp.data != nullptr && p.kl_coef != 0.f) {
    const float diff = p.ref_lp.at(b, s) - q, grow = expm1f(diff);
    r.loss += p.kl_coef * (grow - diff);
    r.a -= p.kl_coef * grow;
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
  const float w = p.weights.data != nullptr ? p.weights.at(b, s) * p.scale : kGrad ? *p.inv_count : 1.f;
  const Gather<kEntropy> g = gather_row<T, NT, kEntropy>(r, z.k, share);
  const float q = (xt - g.zmax) * z.inv_t - logf(g.s), H = kEntropy ? logf(g.s) - kLn2 * g.w / g.s : 0.f;
  const PolicyRow l = policy_row(p, b, s, q, H, w);
  if (threadIdx.x == 0) {
    p.log_probs[row] = q;
    p.losses[row] = l.loss;
    if constexpr (kGrad) {
      p.dlp[row] = l.a;
      if constexpr (kEntropy) { p.dentropy[row] = l.b; p.entropy[row] = H; }
      p.max_sum[row] = f32x2{g.m, g.s};
    }
  }
  if constexpr (kGrad) write_gradient<T, NT, kEntropy>(r, d, slope<kEntropy>(l.a, l.b, g.s, H, z.inv_t), z.k, g.m, static_cast<int>(t));
}

// ---- sums over rows: one workgroup, in double and in a fixed order
constexpr int kSumThreads = 1024, kSumWaves = kSumThreads / kWave;
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

// count: inv_count = scale / max(rows that count, 1); with `loss`: the sum of the losses, times that where they are not weighted yet
__global__ __launch_bounds__(kSumThreads) void policy_sum_kernel(const TokenArgs targets, const float* __restrict__ losses, float* __restrict__ loss,
                                                                 float* __restrict__ inv_count, float scale, int count, int unweighted,
                                                                 int64_t rows, int seq, int vocab, int64_t ignore_index) {
  __shared__ double red_s[kSumWaves];
  __shared__ int red_n[kSumWaves];
  double sum = 0;
  int n = 0;
  for (int64_t row = threadIdx.x; row < rows; row += kSumThreads) {
    if (count) {
      const int64_t b = row / seq;
      n += is_token(targets.at(b, row - b * seq), ignore_index, vocab);
    }
    if (loss != nullptr) sum += losses[row];
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
      for (int s = wave % team * kWave + lane; s < seq; s += team * kWave) {
        sum += p.log_probs[static_cast<int64_t>(b) * seq + s];
        if (p.average) n += is_token(targets.at(b, s), ignore_index, vocab);
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
// the narrowest workgroup that has a row in eight pieces a thread: in a wider one most lanes of a short row would idle
template <typename Fn>
void with_threads(int64_t vocab, int vec, const Fn& fn) {
  const int64_t pieces = (vocab + vec - 1) / vec;
  if (pieces <= 64 * 4) fn(std::integral_constant<int, 64>());
  else if (pieces <= 128 * 4) fn(std::integral_constant<int, 128>());
  else if (pieces <= 256 * 8) fn(std::integral_constant<int, 256>());
  else fn(std::integral_constant<int, 512>());
}
template <typename Fn>
void with_type(const pico_logits& z, const Fn& fn) {
  if (z.dtype == PICO_BF16) with_threads(z.vocab, 8, [&](auto nt) { fn(__bf16(), nt); });
  else with_threads(z.vocab, 4, [&](auto nt) { fn(float(), nt); });
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
  if (z->batch < 0 || z->seq < 0 || z->vocab <= 0 || z->vocab > kMost / 2 || z->seq > kMost || z->batch > kMost || z->batch * z->seq > kMost)
    return fail(PICO_ERR_SHAPE, "%s: batch=%lld seq=%lld vocab=%lld", fn, static_cast<long long>(z->batch), static_cast<long long>(z->seq),
                static_cast<long long>(z->vocab));
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
TokenArgs args(const pico_tokens& t) { return {t.data, t.batch_stride, t.row_stride}; }
ValueArgs args(const pico_values* v) { return v ? ValueArgs{v->data, v->batch_stride, v->row_stride} : ValueArgs{nullptr, 0, 0}; }

int run_log_probs(const char* fn, const pico_logits& z, const pico_tokens& targets, float* log_probs, float* entropy, float* max_sum,
                  float temperature, int64_t ignore_index, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(z.batch * z.seq));
  with_type(z, [&](auto type, auto nt) {
    with_flag(entropy != nullptr, [&](auto with) {
      hipLaunchKernelGGL((log_probs_kernel<decltype(type), decltype(nt)::value, decltype(with)::value>), grid, dim3(decltype(nt)::value), 0, s, args(z, temperature),
                         args(targets), log_probs, entropy, reinterpret_cast<f32x2*>(max_sum), ignore_index);
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
  // (with the gradient at hand the launch usually only looks at grad_out: few workgroups, which walk the rows if they must)
  const dim3 grid(static_cast<unsigned>(have_unit ? std::min<int64_t>(rows, 1024) : rows));
  with_type(*logits, [&](auto type, auto nt) {
    with_flag(with_entropy, [&](auto with) {
      hipLaunchKernelGGL((log_probs_grad_kernel<decltype(type), decltype(nt)::value, decltype(with)::value>), grid, dim3(decltype(nt)::value), 0, static_cast<hipStream_t>(stream),
                         args(*logits, temperature), args(*targets), reinterpret_cast<const f32x2*>(max_sum), entropy, args(dlog_probs), args(dentropy),
                         grad_out, have_unit, static_cast<decltype(type)*>(dlogits), dbatch_stride, drow_stride, rows, ignore_index);
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
    hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(kSumThreads), 0, s, args(*targets), losses, to, inv_count, policy->scale, !weighted,
                       !weighted && !dlogits, rows, static_cast<int>(std::max<int64_t>(logits->seq, 1)), static_cast<int>(logits->vocab), ignore_index);
  };
  if (rows > 0) {
    if (dlogits && !weighted) sum(nullptr);   // the gradient needs scale / count
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
    with_type(*logits, [&](auto type, auto nt) {
      with_flag(with_entropy, [&](auto with) {
        with_flag(dlogits != nullptr, [&](auto grad) {
          hipLaunchKernelGGL((policy_kernel<decltype(type), decltype(nt)::value, decltype(with)::value, decltype(grad)::value>), grid, dim3(decltype(nt)::value), 0, s,
                             args(*logits, temperature), args(*targets), p, static_cast<decltype(type)*>(dlogits), dbatch_stride, drow_stride, ignore_index);
        });
      });
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
