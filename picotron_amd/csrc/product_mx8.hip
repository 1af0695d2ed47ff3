// C = A B^T of rows in the 8-bit form (mx8.h) in bf16: the products of a layer whose activations and weights are held that way.
//
// The matrix instructions with scales multiply 32 e4m3 values of a row by 32 of another and apply both blocks' scales; four (16 x 16 x 128) or two
// (32 x 32 x 64) blocks to an instruction.  Where a lane's values lie: bytes 16 h .. + 15 of the row's 128 (64) and as many from the middle on, h the lane's quarter
// (half) of the wave; its scale is that of block h.  The sums are fp32 registers, but within an instruction the products are added with about 17 bits behind the
// largest: over normal values 1.5e-5 of the result's root mean square (7e-5 with outliers of 20), without a bias and without growth from a contraction
// of 128 to one of 8192.  The rounding of the result to bf16 is 1.7e-3, so the result is bf16 only.
#include "mx8.h"
#include "product_large.h"

namespace pico {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;

struct Mx8Params {
  const uint8_t *a, *b;        // [M, K], [N, K]
  const uint8_t *sa, *sb;      // their scales
  __bf16* c;                   // [M, N rounded up to 8]
  int M, N, K;
};

__device__ __forceinline__ i32x8 both(u32x4 low, u32x4 high) {
  return __builtin_bit_cast(i32x8, __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7));
}

// ---- few rows: MT x NT tiles of 16 x 16 to a workgroup, whose W waves take every W-th 128 of the contraction straight from memory and join their sums in LDS.
template <int MT, int NT, int W>
__global__ __launch_bounds__(W * kWave) void product_mx8_few_kernel(const Mx8Params p) {
  __shared__ f32x4 sums[W][MT * NT][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, n = lane % 16, h = lane / 16;
  const int m0 = blockIdx.y * 16 * MT, n0 = blockIdx.x * 16 * NT, steps = (p.K + kGroup - 1) / kGroup;
  // rows past the matrix read its last one, and what they give is not written
  int64_t ra[MT], rb[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) ra[i] = min(m0 + 16 * i + n, p.M - 1);
#pragma unroll
  for (int j = 0; j < NT; ++j) rb[j] = min(n0 + 16 * j + n, p.N - 1);
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto fragment = [&](const uint8_t* m, int64_t row, int k) __attribute__((always_inline)) {   // (zeros past the contraction, in pieces of 16)
    const uint8_t* at = m + row * p.K + k + 16 * h;
    const u32x4 zero = {0, 0, 0, 0};
    const u32x4 low = k + 16 * h < p.K ? *reinterpret_cast<const u32x4*>(at) : zero, high = k + 64 + 16 * h < p.K ? *reinterpret_cast<const u32x4*>(at + 64) : zero;
    return both(low, high);
  };
#pragma unroll 2
  for (int t = wave; t < steps; t += W) {
    i32x8 fa[MT], fb[NT];
    int sa[MT], sb[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      fb[j] = fragment(p.b, rb[j], t * kGroup);
      sb[j] = p.sb[(static_cast<int64_t>(t) * p.N + rb[j]) * 4 + h];
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      fa[i] = fragment(p.a, ra[i], t * kGroup);
      sa[i] = p.sa[(static_cast<int64_t>(t) * p.M + ra[i]) * 4 + h];
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)   // C^T: a lane holds four columns of a row of C
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa[i], acc[i][j], 0, 0, 0, sb[j], 0, sa[i]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) sums[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
  const int ldc = (p.N + 7) / 8 * 8;
  for (int tile = wave; tile < MT * NT; tile += W) {
    f32x4 v = sums[0][tile][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += sums[w][tile][lane];
    const int row = m0 + 16 * (tile / NT) + n, col = n0 + 16 * (tile % NT) + 4 * h;
    if (row >= p.M || col >= ldc) continue;
    bf16x4 o;   // (columns from N on are 0)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = static_cast<__bf16>(col + e < p.N ? v[e] : 0.f);
    *reinterpret_cast<bf16x4*>(p.c + static_cast<int64_t>(row) * ldc + col) = o;
  }
}

template <int MT, int NT, int W>
void launch_few(const Mx8Params& p, hipStream_t s) {
  hipLaunchKernelGGL((product_mx8_few_kernel<MT, NT, W>), dim3((p.N + 16 * NT - 1) / (16 * NT), (p.M + 16 * MT - 1) / (16 * MT)), dim3(W * kWave), 0, s, p);
}

}  // namespace
}  // namespace pico

using namespace pico;

extern "C" int pico_mx8_product(const pico_mx8* a, const pico_mx8* b, void* c, int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "pico_mx8_product";
  if (int rc = check_mx8_shape(fn, M, K)) return rc;
  if (int rc = check_mx8_shape(fn, N, K)) return rc;
  if (M == 0 || N == 0) return PICO_OK;
  if (int rc = check_mx8(fn, "a", a)) return rc;
  if (int rc = check_mx8(fn, "b", b)) return rc;
  if (!c) return fail(PICO_ERR_NULL, "%s: c is required", fn);
  if (!aligned16(c)) return fail(PICO_ERR_ALIGN, "%s: c must be 16-byte aligned", fn);
  const Mx8Params p = {static_cast<const uint8_t*>(a->data), static_cast<const uint8_t*>(b->data), static_cast<const uint8_t*>(a->scales), static_cast<const uint8_t*>(b->scales),
                       static_cast<__bf16*>(c), (int)M, (int)N, (int)K};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (M <= 16) launch_few<1, 1, 4>(p, s);
  else launch_few<2, 2, 4>(p, s);
  return check_launch(fn);
}

extern "C" int64_t pico_mx8_product_workspace_bytes(int64_t M, int64_t N, int64_t K) { return 0; }
