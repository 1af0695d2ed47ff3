// What makes the 8-bit form (mx8.h) and reads it back beside the products: rows of a tensor, RMSNorm (with the residual's addition) that writes nothing
// else, SwiGLU whose output or checkpoint is held that way and its gradient from that checkpoint.
//
// All of them are bound by memory; each value passes the registers once, and a block's largest value is found among the 4 (bf16) or 8
// (fp32) lanes that hold it.  Measured in bf16, beside 5.1 - 5.4 TB/s of a large copy: rows [16384, 4096] made 37 us (5.5 TB/s), read back 33 (6.1);
// RMSNorm with the residual [16384, 2048] 42 (5.6); SwiGLU [16384, 8192] with its checkpoint 183 (5.9), its gradient 185 (5.8).  More
// groups to a thread, 16 values to a lane and loads past the caches all measured the same.
#include "mx8.h"

namespace pico {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float sigmoid_fast(float x) { return __builtin_amdgcn_rcpf(1.f + fast_exp2(-x * kLog2e)); }

// n / d for n under 2^31: (high half of n m + n) >> s
struct Divide {
  uint32_t m, s, d;
};
Divide divide_by(uint32_t d) {
  uint32_t s = 0;
  while ((uint64_t{1} << s) < d) ++s;
  return {static_cast<uint32_t>((uint64_t{1} << 32) * ((uint64_t{1} << s) - d) / d + 1), s, d};
}
__device__ __forceinline__ uint32_t quotient(uint32_t n, Divide by) { return (__umulhi(n, by.m) + n) >> by.s; }

// Where a thread of the kernels that walk groups of 128 columns stands.  128 / V neighbouring lanes hold a group; the last of a row may be cut short, its
// lanes past the row stay on.
struct Place {
  int64_t row;
  int col, t;      // t: the group in its row
  bool live;
};
template <int V>
__device__ __forceinline__ bool place(Place& p, int64_t groups, Divide per_row, int cols) {
  constexpr int kLanes = kGroup / V;
  const int64_t g = static_cast<int64_t>(blockIdx.x) * (kThreads / kLanes) + threadIdx.x / kLanes;
  if (g >= groups) return false;
  const uint32_t row = quotient(static_cast<uint32_t>(g), per_row);
  p.row = row;
  p.t = static_cast<int>(static_cast<uint32_t>(g) - row * per_row.d);
  p.col = p.t * kGroup + static_cast<int>(threadIdx.x % kLanes) * V;
  p.live = p.col < cols;
  return true;
}
template <int V>
__device__ __forceinline__ void store_block(const pico_mx8& y, const Place& p, int64_t rows, int cols, const float (&v)[V]) {
  const Codes<V> c = encode<V>(v);
  const uint32_t scales = four_scales<V>(c.scale, threadIdx.x);
  if (!p.live) return;
  store_codes<V>(static_cast<uint8_t*>(y.data) + p.row * cols + p.col, c.word);
  if (threadIdx.x % (kGroup / V) == 0) static_cast<uint32_t*>(y.scales)[p.t * rows + p.row] = scales;
}
template <int V>
__device__ __forceinline__ void load_block(const pico_mx8& x, const Place& p, int64_t rows, int cols, float (&v)[V]) {
  uint32_t word[V / 4];
  load_codes<V>(static_cast<const uint8_t*>(x.data) + p.row * cols + p.col, word);
  decode<V>(word, static_cast<const uint8_t*>(x.scales)[(p.t * rows + p.row) * 4 + p.col % kGroup / kBlock], v);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const T* __restrict__ x, const pico_mx8 y, int64_t rows, int cols, int64_t ld, int64_t groups, Divide per_row) {
  constexpr int V = io<T>::kVec;
  Place p;
  if (!place<V>(p, groups, per_row, cols)) return;
  float v[V] = {};
  if (p.live) io<T>::load(x + p.row * ld + p.col, v);
  store_block<V>(y, p, rows, cols, v);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const pico_mx8 x, T* __restrict__ y, int64_t rows, int cols, int64_t ld, int64_t groups, Divide per_row) {
  constexpr int V = io<T>::kVec;
  Place p;
  if (!place<V>(p, groups, per_row, cols) || !p.live) return;
  float v[V];
  load_block<V>(x, p, rows, cols, v);
  io<T>::store(y + p.row * ld + p.col, v);
}

// silu(gate) * up; y and y8, either or both, and the checkpoint where it is wanted
template <typename T>
__global__ __launch_bounds__(kThreads) void swiglu_mx8_fwd_kernel(const T* __restrict__ gate, const T* __restrict__ up, T* __restrict__ y, const pico_mx8 y8,
                                                                  const pico_mx8 gate8, const pico_mx8 up8, int64_t rows, int cols, int64_t gate_ld, int64_t up_ld,
                                                                  int64_t groups, Divide per_row) {
  constexpr int V = io<T>::kVec;
  Place p;
  if (!place<V>(p, groups, per_row, cols)) return;
  float g[V] = {}, u[V] = {}, o[V];
  if (p.live) {
    io<T>::load(gate + p.row * gate_ld + p.col, g);
    io<T>::load(up + p.row * up_ld + p.col, u);
  }
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = g[e] * sigmoid_fast(g[e]) * u[e];
  if (gate8.data != nullptr) {
    store_block<V>(gate8, p, rows, cols, g);
    store_block<V>(up8, p, rows, cols, u);
  }
  if (y8.data != nullptr) store_block<V>(y8, p, rows, cols, o);
  if (y != nullptr && p.live) io<T>::store(y + p.row * cols + p.col, o);
}

// With g, u what the checkpoint stands for and s = sigmoid(g): dgate = dy u s (1 + g (1 - s)), dup = dy g s; y = g s u again where it is wanted.
// kFrom: dy of rows of pitch dy_ld; or contiguous, in fp32 and in `parts` pieces to be added, as a product leaves it; or contiguous in 20 bits.  [8192, 11008] 145, 184
// and 150 us, a copy's rate.
enum class Upstream { Rows, Sums, Bits20 };
template <typename T, Upstream kFrom>
__global__ __launch_bounds__(kThreads) void swiglu_mx8_bwd_kernel(const std::conditional_t<kFrom == Upstream::Sums, float, T>* __restrict__ dy, const uint32_t* __restrict__ dy_left, int parts, const pico_mx8 gate8, const pico_mx8 up8, T* __restrict__ dgate, T* __restrict__ dup,
                                                                  T* __restrict__ y, int64_t rows, int cols, int64_t dy_ld, int64_t dgate_ld, int64_t dup_ld, int64_t groups,
                                                                  Divide per_row) {
  constexpr int V = io<T>::kVec;
  Place p;
  if (!place<V>(p, groups, per_row, cols) || !p.live) return;
  float d[V], g[V], u[V], dg[V], du[V], o[V];
  load_block<V>(gate8, p, rows, cols, g);
  load_block<V>(up8, p, rows, cols, u);
  if constexpr (kFrom == Upstream::Sums) {
    const float* from = dy + p.row * cols + p.col;
    f32x4 sum[V / 4];
#pragma unroll
    for (int q = 0; q < V / 4; ++q) sum[q] = *reinterpret_cast<const f32x4*>(from + 4 * q);
    for (int i = 1; i < parts; ++i) {
      from += rows * cols;
#pragma unroll
      for (int q = 0; q < V / 4; ++q) sum[q] += *reinterpret_cast<const f32x4*>(from + 4 * q);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) d[e] = sum[e / 4][e % 4];
  } else if constexpr (kFrom == Upstream::Bits20) {
    const int64_t at = p.row * cols + p.col;
    const u32x4 raw = *reinterpret_cast<const u32x4*>(dy + at);
    const uint32_t word = dy_left[at / 8];
#pragma unroll
    for (int e = 0; e < V; ++e) d[e] = from_bits20(e % 2 ? raw[e / 2] & 0xffff0000u : raw[e / 2] << 16, word, e);
  } else {
    io<T>::load(dy + p.row * dy_ld + p.col, d);
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float s = sigmoid_fast(g[e]), gs = g[e] * s;
    dg[e] = d[e] * u[e] * s * (1.f + g[e] * (1.f - s));
    du[e] = d[e] * gs;
    o[e] = gs * u[e];
  }
  io<T>::store(dgate + p.row * dgate_ld + p.col, dg);
  io<T>::store(dup + p.row * dup_ld + p.col, du);
  if (y != nullptr) io<T>::store(y + p.row * cols + p.col, o);
}

// ---- RMSNorm: y = (x + residual) rstd w in the 8-bit form only
template <int G>
__device__ __forceinline__ double group_sum(double v, double* smem) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  if constexpr (G == kWave) {
    return v;
  } else {
    if (threadIdx.x % kWave == 0) smem[threadIdx.x / kWave] = v;
    __syncthreads();
    double t = 0.;
#pragma unroll
    for (int i = 0; i < G / kWave; ++i) t += smem[i];
    return t;
  }
}

// Whether what an fp32 value stands for, up to 4 of its last places away (three roundings, and that of h in fp32), may lie in the middle of two codes: its last 19 bits are 0 there.
// This is under kNearMiddle then.
constexpr uint32_t kNearMiddle = (8u << 13) + 1;
__device__ __forceinline__ uint32_t past_a_middle(float v) { return (__float_as_uint(v) << 13) + (4u << 13); }
// y in 32 bits, the last one 1 where they do not hold it: no such value lies in the middle of two codes
__device__ __forceinline__ float no_middle(double y) {
  const float s = static_cast<float>(y);
  const double left = y - s;
  const int bits = __float_as_int(s), away = (left < 0.) == (bits < 0) ? 1 : -1;
  return __int_as_float(fabs(left) > 0. && bits % 2 == 0 ? bits + away : bits);
}

// of eight values
__device__ __forceinline__ uint32_t bf16_left(const float (&v)[8]) {
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) word |= pico::bf16_left(v[e]) << (4 * e);
  return word;
}

// A row to a wave (G 64) or to the workgroup, NV pieces of 16 bytes to a thread, which stay in registers between the sum of squares and the output; four at most, that a row is
// requested as a whole ([13986, 9984] in bf16 266 us by 256 threads with eight, 187 by 1024 with two).
// Every code is that of the exact value.  Beside the middle of two codes an error of 2^-24 would take the other one, so the sum of squares is in 64 bits, with what x + residual loses in 32,
// and pieces with such a value are made once more in 64 bits and written over ([16384, 2048] with the residual 42 us, as without any of it; 22.8 for 22.3 where there is none).  A
// kernel for each: without a residual's registers 76 of them, five waves to a SIMD, where one kernel for both takes 98 and 25.2 us.
constexpr int norm_threads(int g) { return g < kThreads ? kThreads : g; }
template <typename T>
__device__ __forceinline__ float value_of(u32x4 raw, int e) {
  if constexpr (std::is_same_v<T, float>) return __uint_as_float(raw[e]);
  else return __uint_as_float(e % 2 ? raw[e / 2] & 0xffff0000u : raw[e / 2] << 16);
}
template <typename T, int G, int NV, bool kRes>
__global__ __launch_bounds__(norm_threads(G)) void rmsnorm_mx8_kernel(const T* __restrict__ x, const T* __restrict__ w, const pico_mx8 y, float* __restrict__ rstd,
                                                               const T* __restrict__ res_in, T* __restrict__ res_out, uint32_t* __restrict__ res_left, int64_t rows, int hidden, float eps, double inv_hidden) {
  Arguments<0, 64>().arrive();
  constexpr int V = io<T>::kVec;
  __shared__ double smem[norm_threads(G) / kWave];
  const int t = threadIdx.x % G, nvec = hidden / V;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (norm_threads(G) / G) + threadIdx.x / G;
  if (row >= rows) return;   // (G over 64: uniform over the workgroup, which meets at a barrier below)
  const int64_t at = row * hidden;
  // everything that the row needs is requested before the first of it is used; pieces past the row re-read its first
  auto piece = [&](int j) { return (t + j * G < nvec ? t + j * G : 0) * V; };
  u32x4 x_raw[NV], r_raw[kRes ? NV : 1], w_raw[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) x_raw[j] = *reinterpret_cast<const u32x4*>(x + at + piece(j));
  if constexpr (kRes) {
#pragma unroll
    for (int j = 0; j < NV; ++j) r_raw[j] = *reinterpret_cast<const u32x4*>(res_in + at + piece(j));
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) w_raw[j] = *reinterpret_cast<const u32x4*>(w + piece(j));
  __builtin_amdgcn_sched_barrier(0);
  float vals[NV][V];
  double ss = 0.;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const bool live = t + j * G < nvec;
    double piece_ss = 0.;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      vals[j][e] = value_of<T>(x_raw[j], e);
      double h = vals[j][e];
      if constexpr (kRes) {
        const float b = value_of<T>(r_raw[j], e);
        vals[j][e] += b;
        h += b;   // (with what the sum in 32 bits loses)
      }
      piece_ss += h * h;
    }
    asm volatile("" : "+v"(piece_ss));   // (here and now: behind the branch that needs it the operands would take 40 registers more)
    if (live) ss += piece_ss;
    if constexpr (kRes) {
      if (res_out != nullptr && live) store_as<T, true>(res_out + at + piece(j), vals[j]);
      if constexpr (V == 8) {
        if (res_left != nullptr && live) res_left[row * nvec + t + j * G] = bf16_left(vals[j]);
      }
    }
  }
  const double mean = group_sum<G>(ss, smem) * inv_hidden + eps;
  float r = rsqrtf(static_cast<float>(mean));
  double root = r;
  if (r > 0.f && r < __builtin_huge_valf()) root += 0.5 * r * (1. - mean * r * r);   // (0: a row with an infinity)
  r = static_cast<float>(root);
  if (rstd != nullptr && t == 0) rstd[row] = r;
  auto put = [&](int v, const float (&o)[V]) {
    const Codes<V> c = encode<V>(o);
    const uint32_t scales = four_scales<V>(v < nvec ? c.scale : 0u, t);
    if (v < nvec) {
      store_codes<V>(static_cast<uint8_t*>(y.data) + at + static_cast<int64_t>(v) * V, c.word);
      if (v % (kGroup / V) == 0) static_cast<uint32_t*>(y.scales)[static_cast<int64_t>(v / (kGroup / V)) * rows + row] = scales;
    }
  };
  uint32_t anew = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = t + j * G;
    if (__builtin_amdgcn_readfirstlane(v) >= nvec) break;   // (uniform: whole waves of pieces past the row)
    float o[V];
    uint32_t nearest = ~0u;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      o[e] = vals[j][e] * r * value_of<T>(w_raw[j], e);
      nearest = min(nearest, past_a_middle(o[e]));
    }
    if (__any(nearest < kNearMiddle)) {
      bool near = false;   // (0 is no such value: rows of padding)
#pragma unroll
      for (int e = 0; e < V; ++e) near |= past_a_middle(o[e]) < kNearMiddle && o[e] != 0.f;
      if (__any(near && v < nvec)) anew |= 1u << j;
    }
    put(v, o);
  }
  // One in a hundred of a wave's pieces, from the operands where they still are (kept in registers until here they would take 90 more).  Where the sum has taken the place of one, the
  // codes stay those of the values in 32 bits.
  if (anew == 0 || (kRes && (res_out == res_in || res_out == x))) return;
  const T *x_again = x, *r_again = res_in;
  asm volatile("" : "+s"(x_again), "+s"(r_again));   // (loads of their own)
#pragma unroll 1
  for (int j = 0; j < NV; ++j) {
    if ((anew >> j & 1) == 0) continue;
    const int v = t + j * G;
    const u32x4 a = *reinterpret_cast<const u32x4*>(x_again + at + piece(j)), gamma = *reinterpret_cast<const u32x4*>(w + piece(j));
    u32x4 b = {};
    if constexpr (kRes) b = *reinterpret_cast<const u32x4*>(r_again + at + piece(j));
    float o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      double h = value_of<T>(a, e);
      if constexpr (kRes) h += value_of<T>(b, e);
      o[e] = no_middle(h * root * value_of<T>(gamma, e));
    }
    put(v, o);
  }
}

template <typename T, int G, int NV>
void launch_norm(const void* x, const void* w, const pico_mx8& y, float* rstd, const void* ri, void* ro, uint32_t* left, int64_t rows, int hidden, float eps, hipStream_t s) {
  constexpr int kRows = norm_threads(G) / G;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((rows + kRows - 1) / kRows)), dim3(norm_threads(G)), 0, s, static_cast<const T*>(x), static_cast<const T*>(w), y, rstd,
                       static_cast<const T*>(ri), static_cast<T*>(ro), left, rows, hidden, eps, 1. / hidden);
  };
  if (ri != nullptr) go(rmsnorm_mx8_kernel<T, G, NV, true>);
  else go(rmsnorm_mx8_kernel<T, G, NV, false>);
}
template <typename T>
void dispatch_norm(const void* x, const void* w, const pico_mx8& y, float* rstd, const void* ri, void* ro, uint32_t* left, int64_t rows, int hidden, float eps, hipStream_t s) {
  const int nvec = hidden / io<T>::kVec;
  if (nvec <= 64) return launch_norm<T, 64, 1>(x, w, y, rstd, ri, ro, left, rows, hidden, eps, s);
  if (nvec <= 128) return launch_norm<T, 64, 2>(x, w, y, rstd, ri, ro, left, rows, hidden, eps, s);
  if (nvec <= 256) return launch_norm<T, 64, 4>(x, w, y, rstd, ri, ro, left, rows, hidden, eps, s);
  if (nvec <= 512) return launch_norm<T, 256, 2>(x, w, y, rstd, ri, ro, left, rows, hidden, eps, s);
  if (nvec <= 1024) return launch_norm<T, 256, 4>(x, w, y, rstd, ri, ro, left, rows, hidden, eps, s);
  if (nvec <= 2048) return launch_norm<T, 1024, 2>(x, w, y, rstd, ri, ro, left, rows, hidden, eps, s);
  launch_norm<T, 1024, 4>(x, w, y, rstd, ri, ro, left, rows, hidden, eps, s);
}

int vec_of(int dtype) { return dtype == PICO_BF16 ? 8 : 4; }
int check_dtype(const char* fn, int dtype) {
  return dtype == PICO_BF16 || dtype == PICO_F32 ? PICO_OK : fail(PICO_ERR_DTYPE, "%s: dtype code %d not supported", fn, dtype);
}
// a tensor of rows of pitch ld beside the 8-bit operands
int check_rows(const char* fn, const char* what, const void* p, int64_t cols, int64_t ld, int dtype) {
  if (!p) return fail(PICO_ERR_NULL, "%s: %s is required", fn, what);
  if (ld < cols) return fail(PICO_ERR_STRIDE, "%s: %s has a row pitch under its columns", fn, what);
  if (!aligned16(p) || ld % vec_of(dtype) != 0) return fail(PICO_ERR_ALIGN, "%s: %s must be 16-byte aligned, its row pitch a multiple of %d", fn, what, vec_of(dtype));
  return PICO_OK;
}
struct Walk {
  int64_t groups;
  Divide per_row;
  dim3 grid;
};
Walk walk(int64_t rows, int64_t cols, int dtype) {
  const int64_t per_row = (cols + kGroup - 1) / kGroup, groups = rows * per_row, per_block = kThreads / (kGroup / vec_of(dtype));
  return {groups, divide_by(static_cast<uint32_t>(per_row)), dim3(static_cast<unsigned>((groups + per_block - 1) / per_block))};
}

}  // namespace
}  // namespace pico

using namespace pico;

#define PICO_TRY(call) \
  if (int rc = (call)) return rc

extern "C" int pico_mx8_quantize(const void* x, const pico_mx8* y, int64_t rows, int64_t cols, int64_t x_ld, int dtype, void* stream) {
  const char* fn = "pico_mx8_quantize";
  PICO_TRY(check_dtype(fn, dtype));
  PICO_TRY(check_mx8_shape(fn, rows, cols));
  if (rows == 0) return PICO_OK;
  PICO_TRY(check_rows(fn, "x", x, cols, x_ld, dtype));
  PICO_TRY(check_mx8(fn, "y", y));
  const Walk w = walk(rows, cols, dtype);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == PICO_BF16)
    hipLaunchKernelGGL(quantize_kernel<__bf16>, w.grid, dim3(kThreads), 0, s, static_cast<const __bf16*>(x), *y, rows, static_cast<int>(cols), x_ld, w.groups, w.per_row);
  else
    hipLaunchKernelGGL(quantize_kernel<float>, w.grid, dim3(kThreads), 0, s, static_cast<const float*>(x), *y, rows, static_cast<int>(cols), x_ld, w.groups, w.per_row);
  return check_launch(fn);
}

extern "C" int pico_mx8_dequantize(const pico_mx8* x, void* y, int64_t rows, int64_t cols, int64_t y_ld, int dtype, void* stream) {
  const char* fn = "pico_mx8_dequantize";
  PICO_TRY(check_dtype(fn, dtype));
  PICO_TRY(check_mx8_shape(fn, rows, cols));
  if (rows == 0) return PICO_OK;
  PICO_TRY(check_mx8(fn, "x", x));
  PICO_TRY(check_rows(fn, "y", y, cols, y_ld, dtype));
  const Walk w = walk(rows, cols, dtype);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == PICO_BF16)
    hipLaunchKernelGGL(dequantize_kernel<__bf16>, w.grid, dim3(kThreads), 0, s, *x, static_cast<__bf16*>(y), rows, static_cast<int>(cols), y_ld, w.groups, w.per_row);
  else
    hipLaunchKernelGGL(dequantize_kernel<float>, w.grid, dim3(kThreads), 0, s, *x, static_cast<float*>(y), rows, static_cast<int>(cols), y_ld, w.groups, w.per_row);
  return check_launch(fn);
}

extern "C" int pico_rmsnorm_mx8_fwd(const void* x, const void* weight, const pico_mx8* y, float* rstd, const void* residual_in, void* residual_out, void* residual_left, int64_t rows,
                                    int64_t hidden, float eps, int dtype, void* stream) {
  const char* fn = "pico_rmsnorm_mx8_fwd";
  PICO_TRY(check_dtype(fn, dtype));
  PICO_TRY(check_mx8_shape(fn, rows, hidden));
  if (hidden > 16384) return fail(PICO_ERR_SHAPE, "%s: hidden=%lld (16384 at most)", fn, (long long)hidden);
  // (a launch's threads: 2^24 - 1 workgroups of 256 with a wave to a row; longer rows take more and are fewer by the check above)
  if (rows > (int64_t{1} << 26) - 4) return fail(PICO_ERR_SHAPE, "%s: rows=%lld (2^26 - 4 at most)", fn, (long long)rows);
  if (rows == 0) return PICO_OK;
  PICO_TRY(check_rows(fn, "x", x, hidden, hidden, dtype));
  PICO_TRY(check_rows(fn, "weight", weight, hidden, hidden, dtype));
  PICO_TRY(check_mx8(fn, "y", y));
  if ((residual_out || residual_left) && !residual_in) return fail(PICO_ERR_NULL, "%s: residual_out or residual_left without residual_in", fn);
  if (residual_left && dtype != PICO_BF16) return fail(PICO_ERR_DTYPE, "%s: residual_left is bf16's", fn);
  if (!aligned16(residual_in) || !aligned16(residual_out) || !aligned16(residual_left)) return fail(PICO_ERR_ALIGN, "%s: pointers must be 16-byte aligned", fn);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == PICO_BF16) dispatch_norm<__bf16>(x, weight, *y, rstd, residual_in, residual_out, static_cast<uint32_t*>(residual_left), rows, static_cast<int>(hidden), eps, s);
  else dispatch_norm<float>(x, weight, *y, rstd, residual_in, residual_out, static_cast<uint32_t*>(residual_left), rows, static_cast<int>(hidden), eps, s);
  return check_launch(fn);
}

extern "C" int pico_swiglu_mx8_fwd(const void* gate, const void* up, void* y, const pico_mx8* y8, const pico_mx8* gate8, const pico_mx8* up8, int64_t rows, int64_t cols,
                                   int64_t gate_ld, int64_t up_ld, int dtype, void* stream) {
  const char* fn = "pico_swiglu_mx8_fwd";
  PICO_TRY(check_dtype(fn, dtype));
  PICO_TRY(check_mx8_shape(fn, rows, cols));
  if (rows == 0) return PICO_OK;
  if (!y && !y8) return fail(PICO_ERR_NULL, "%s: y or y8 is required", fn);
  if (!gate8 != !up8) return fail(PICO_ERR_NULL, "%s: gate8 and up8 come together", fn);
  PICO_TRY(check_rows(fn, "gate", gate, cols, gate_ld, dtype));
  PICO_TRY(check_rows(fn, "up", up, cols, up_ld, dtype));
  if (y) PICO_TRY(check_rows(fn, "y", y, cols, cols, dtype));
  if (y8) PICO_TRY(check_mx8(fn, "y8", y8));
  if (gate8) {
    PICO_TRY(check_mx8(fn, "gate8", gate8));
    PICO_TRY(check_mx8(fn, "up8", up8));
  }
  const Walk w = walk(rows, cols, dtype);
  const pico_mx8 none = {nullptr, nullptr};
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto kernel, auto zero) {
    using T = decltype(zero);
    hipLaunchKernelGGL(kernel, w.grid, dim3(kThreads), 0, s, static_cast<const T*>(gate), static_cast<const T*>(up), static_cast<T*>(y), y8 ? *y8 : none, gate8 ? *gate8 : none,
                       up8 ? *up8 : none, rows, static_cast<int>(cols), gate_ld, up_ld, w.groups, w.per_row);
  };
  if (dtype == PICO_BF16) go(swiglu_mx8_fwd_kernel<__bf16>, __bf16());
  else go(swiglu_mx8_fwd_kernel<float>, float());
  return check_launch(fn);
}

extern "C" int pico_swiglu_mx8_bwd(const void* dy, const pico_mx8* gate8, const pico_mx8* up8, void* dgate, void* dup, void* y, int64_t rows, int64_t cols, int64_t dy_ld,
                                   int64_t dgate_ld, int64_t dup_ld, int dtype, void* stream) {
  const char* fn = "pico_swiglu_mx8_bwd";
  PICO_TRY(check_dtype(fn, dtype));
  PICO_TRY(check_mx8_shape(fn, rows, cols));
  if (rows == 0) return PICO_OK;
  PICO_TRY(check_rows(fn, "dy", dy, cols, dy_ld, dtype));
  PICO_TRY(check_mx8(fn, "gate8", gate8));
  PICO_TRY(check_mx8(fn, "up8", up8));
  PICO_TRY(check_rows(fn, "dgate", dgate, cols, dgate_ld, dtype));
  PICO_TRY(check_rows(fn, "dup", dup, cols, dup_ld, dtype));
  if (y) PICO_TRY(check_rows(fn, "y", y, cols, cols, dtype));
  const Walk w = walk(rows, cols, dtype);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto kernel, auto zero) {
    using T = decltype(zero);
    hipLaunchKernelGGL(kernel, w.grid, dim3(kThreads), 0, s, static_cast<const T*>(dy), nullptr, 1, *gate8, *up8, static_cast<T*>(dgate), static_cast<T*>(dup), static_cast<T*>(y), rows,
                       static_cast<int>(cols), dy_ld, dgate_ld, dup_ld, w.groups, w.per_row);
  };
  if (dtype == PICO_BF16) go(swiglu_mx8_bwd_kernel<__bf16, Upstream::Rows>, __bf16());
  else go(swiglu_mx8_bwd_kernel<float, Upstream::Rows>, float());
  return check_launch(fn);
}

namespace {
// of bf16, from a contiguous dy that holds more than that
template <Upstream kFrom, typename From>
int swiglu_bwd_from(const char* fn, const From* dy, const void* dy_left, int parts, const pico_mx8* gate8, const pico_mx8* up8, void* dgate, void* dup, void* y, int64_t rows, int64_t cols,
                    int64_t dgate_ld, int64_t dup_ld, void* stream) {
  PICO_TRY(check_mx8_shape(fn, rows, cols));
  if (parts < 1 || parts > 64) return fail(PICO_ERR_SHAPE, "%s: %d pieces (1 .. 64)", fn, parts);
  if (rows == 0) return PICO_OK;
  PICO_TRY(check_rows(fn, "dy", dy, cols, cols, kFrom == Upstream::Sums ? PICO_F32 : PICO_BF16));
  if (kFrom == Upstream::Bits20) PICO_TRY(check_rows(fn, "dy_left", dy_left, cols, cols, PICO_F32));
  PICO_TRY(check_mx8(fn, "gate8", gate8));
  PICO_TRY(check_mx8(fn, "up8", up8));
  PICO_TRY(check_rows(fn, "dgate", dgate, cols, dgate_ld, PICO_BF16));
  PICO_TRY(check_rows(fn, "dup", dup, cols, dup_ld, PICO_BF16));
  if (y) PICO_TRY(check_rows(fn, "y", y, cols, cols, PICO_BF16));
  const Walk w = walk(rows, cols, PICO_BF16);
  hipLaunchKernelGGL((swiglu_mx8_bwd_kernel<__bf16, kFrom>), w.grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), dy, static_cast<const uint32_t*>(dy_left), parts, *gate8, *up8,
                     static_cast<__bf16*>(dgate), static_cast<__bf16*>(dup), static_cast<__bf16*>(y), rows, static_cast<int>(cols), cols, dgate_ld, dup_ld, w.groups, w.per_row);
  return check_launch(fn);
}
}  // namespace

extern "C" int pico_swiglu_mx8_bwd_sums(const float* dy, int parts, const pico_mx8* gate8, const pico_mx8* up8, void* dgate, void* dup, void* y, int64_t rows, int64_t cols, int64_t dgate_ld,
                                        int64_t dup_ld, void* stream) {
  return swiglu_bwd_from<Upstream::Sums>("pico_swiglu_mx8_bwd_sums", dy, nullptr, parts, gate8, up8, dgate, dup, y, rows, cols, dgate_ld, dup_ld, stream);
}
extern "C" int pico_swiglu_mx8_bwd_bits20(const void* dy, const void* dy_left, const pico_mx8* gate8, const pico_mx8* up8, void* dgate, void* dup, void* y, int64_t rows, int64_t cols,
                                        int64_t dgate_ld, int64_t dup_ld, void* stream) {
  return swiglu_bwd_from<Upstream::Bits20>("pico_swiglu_mx8_bwd_bits20", static_cast<const __bf16*>(dy), dy_left, 1, gate8, up8, dgate, dup, y, rows, cols, dgate_ld, dup_ld, stream);
}
